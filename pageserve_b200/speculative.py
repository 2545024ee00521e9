"""Decoding with trees of drafted tokens over the paged cache.

The reference feeds one token per sequence and decode step
(engine/runner.py:65-79). Here a step may verify several drafted continuations
of every sequence at once: the new tokens of a request form a tree (row 0, the
root, is its last confirmed token; every other row's parent is an earlier row
of the request), each row is stored in the cache at ``seq_len + row`` and sees
the request's cached tokens and its own ancestors.

* :func:`build_step_tables` makes a step's block tables, positions, KV slots
  and ancestor masks on the device, from lengths that live there and a list of
  free blocks (the block bookkeeping of engine/scheduler.py without a host
  round trip); it serves ordinary decode and prefill steps too.
* :func:`tree_attention` is :func:`pageserve_b200.paged_attention.paged_attention`
  with the tree's rule in place of the causal one.
* :func:`accept_trees` finds the longest path that the model's own next tokens
  agree with and moves its keys and values to the positions they keep.

``PagedCausalLM.verify_trees`` runs the three around one model pass. All
lengths stay on the device, so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .paged_attention import AttentionWorkspace

MAX_NODES = 256  # tree nodes per request


class StepTables(NamedTuple):
    """A step's device metadata (int32; ``tree_mask`` int64)."""
    block_tables: torch.Tensor  # (B, max_blocks), -1 behind a request's blocks
    held: torch.Tensor          # (B,) entries each row now has
    cu_q: torch.Tensor          # (B + 1,) row offsets
    positions: torch.Tensor     # (total_tokens,) rotary positions
    slots: torch.Tensor         # (total_tokens,) cache slots, -1: none
    tree_mask: torch.Tensor | None  # (total_tokens, ceil(max_q_len / 64)) ancestor bits; None without parents
    free_used: torch.Tensor     # (1,) blocks the step wants from the free list


class Accepted(NamedTuple):
    """What a verified step keeps (int32)."""
    num: torch.Tensor        # (B,) accepted nodes, the root among them
    nodes: torch.Tensor      # (B, max_q_len) the path's rows, -1 behind
    tokens: torch.Tensor     # (B, max_q_len) the tokens the step yields, -1 behind
    start_pos: torch.Tensor  # (B,) tokens in the cache after the step


def _int32(name: str, device: torch.device, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError(f"{name}: metadata must be contiguous int32")
        if t.device != device:
            raise ValueError(f"{name}: tensors on different devices ({t.device}, {device})")


def _mask_words(name: str, tree_mask: torch.Tensor, rows: int, max_q_len: int, device: torch.device) -> None:
    if tree_mask.dtype != torch.int64 or not tree_mask.is_contiguous():
        raise TypeError(f"{name}: tree_mask must be contiguous int64")
    if tree_mask.device != device:
        raise ValueError(f"{name}: tensors on different devices ({tree_mask.device}, {device})")
    if tree_mask.dim() != 2 or tree_mask.shape[0] < rows or tree_mask.shape[1] != (max_q_len + 63) // 64:
        raise ValueError(f"{name}: tree_mask {tuple(tree_mask.shape)} does not hold {rows} rows of "
                         f"{(max_q_len + 63) // 64} words")


def build_step_tables(seq_lens: torch.Tensor, q_lens: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
                      free_blocks: torch.Tensor, num_blocks: int, block_size: int, total_tokens: int,
                      parents: torch.Tensor | None = None, max_q_len: int | None = None,
                      out: torch.Tensor | None = None) -> StepTables:
    """Block tables, positions, slots and ancestor masks of one step.

    seq_lens, q_lens, held int32 (B,): each request's cached tokens, new tokens
    (0: it waits) and blocks in its row of block_tables int32 (B, max_blocks).
    Missing blocks are taken from free_blocks int32 (F,) in request order.
    total_tokens: the step's rows (at least the sum of q_lens; the rows behind
    get position 0, slot -1). parents int32 (total_tokens,): each row's parent
    among its request's rows, -1 for none; a row's position is then its depth
    past seq_len, and tree_mask is made (max_q_len bounds q_lens, at most
    256). Without parents the rows are a chunk at seq_len + i. ``out`` takes
    the tables; it may be block_tables itself. A free list that is too short
    leaves -1 entries and slots, free_used above F and device error 6; lengths
    beyond the given bounds are device error 5 (``_lib.raise_on_device_error``)."""
    _lib.require_cuda(seq_lens, q_lens, block_tables, held, free_blocks, parents, out)
    dev = seq_lens.device
    _int32("build_step_tables", dev, seq_lens, q_lens, block_tables, held, free_blocks)
    B = seq_lens.numel()
    if B == 0:
        raise ValueError("build_step_tables: empty batch")
    if block_tables.dim() != 2 or block_tables.shape[0] != B or q_lens.numel() != B or held.numel() != B:
        raise ValueError("build_step_tables: q_lens, held and block_tables need one entry per request")
    width = block_tables.shape[1]
    if out is None:
        tables = torch.empty_like(block_tables)
    else:
        _int32("build_step_tables", dev, out)
        if out.shape != block_tables.shape:
            raise ValueError("build_step_tables: out must have block_tables' shape")
        tables = out
    T = int(total_tokens)
    if T < 0:
        raise ValueError("build_step_tables: total_tokens below 0")
    mask = None
    if parents is not None:
        _int32("build_step_tables", dev, parents)
        if parents.numel() < T:
            raise ValueError(f"build_step_tables: {parents.numel()} parents for {T} rows")
        if max_q_len is None:
            raise ValueError("build_step_tables: max_q_len bounds the trees; pass it with parents")
        mask = torch.empty((T, (max_q_len + 63) // 64), dtype=torch.int64, device=dev)
    # one allocation for the small int32 outputs
    buf = torch.empty(2 * B + 2 + 2 * T, dtype=torch.int32, device=dev)
    held_out, cu_q, used, positions, slots = buf.split([B, B + 1, 1, T, T])
    with torch.cuda.device(dev):
        _lib.check(_lib.load().ps_build_step_tables(
            tables.data_ptr(), held_out.data_ptr(), cu_q.data_ptr(), positions.data_ptr(), slots.data_ptr(),
            _lib.ptr(mask), used.data_ptr(), block_tables.data_ptr(), held.data_ptr(), seq_lens.data_ptr(),
            q_lens.data_ptr(), free_blocks.data_ptr(), _lib.ptr(parents), B, T, max_q_len or 0, width,
            free_blocks.numel(), num_blocks, block_size, _lib.stream_ptr(dev)), "build_step_tables")
    return StepTables(tables, held_out, cu_q, positions, slots, mask, used)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                   cu_q: torch.Tensor, start_pos: torch.Tensor, tree_mask: torch.Tensor, max_q_len: int, max_ctx: int,
                   out: torch.Tensor | None = None, workspace: AttentionWorkspace | None = None) -> torch.Tensor:
    """Paged attention of drafted trees: q (total_q, Hq, D), caches (NB, bs,
    Hkv, D), tables, cu_q and start_pos as in ``paged_attention``; tree_mask
    int64 (total_q, ceil(max_q_len / 64)) from :func:`build_step_tables`.
    Node i of request b sees the cached keys [0, start_pos[b]) and the nodes
    of its mask row (stored at start_pos[b] + node); 0 when it sees nothing.
    Rows of ``out`` behind cu_q[-1] are left as they were. A workspace serves
    calls on one stream at a time; without one the scratch is allocated per
    call."""
    _lib.require_cuda(q, k_cache, v_cache, block_tables, cu_q, start_pos, tree_mask, out)
    if q.dim() != 3 or k_cache.dim() != 4 or block_tables.dim() != 2:
        raise ValueError("tree_attention: q (T, Hq, D), caches (NB, bs, Hkv, D), block_tables (B, max_blocks)")
    dev = q.device
    total_q, hq, d = q.shape
    nb, bs, hkv, d2 = k_cache.shape
    if d2 != d or v_cache.shape != k_cache.shape:
        raise ValueError("tree_attention: cache / query head_dim mismatch")
    if q.dtype != k_cache.dtype or q.dtype != v_cache.dtype:
        raise TypeError("tree_attention: q and cache dtypes differ")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("tree_attention: the caches must be contiguous")
    if k_cache.device != dev or v_cache.device != dev:
        raise ValueError("tree_attention: tensors on different devices")
    _int32("tree_attention", dev, block_tables, cu_q, start_pos)
    B = start_pos.numel()
    if block_tables.shape[0] != B or cu_q.numel() != B + 1:
        raise ValueError("tree_attention: block_tables, cu_q and start_pos disagree on the batch")
    _mask_words("tree_attention", tree_mask, total_q, max_q_len, dev)
    q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("tree_attention: out must be contiguous, with q's shape, dtype and device")
    lib = _lib.load()
    nbytes = lib.ps_tree_attention_workspace_size(B, max_q_len, max_ctx, hq, hkv, d)
    buf = (workspace or AttentionWorkspace()).get(nbytes, dev)
    with torch.cuda.device(dev):
        _lib.check(lib.ps_tree_attention(out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                         block_tables.data_ptr(), block_tables.shape[1], cu_q.data_ptr(),
                                         start_pos.data_ptr(), tree_mask.data_ptr(), B, total_q, max_q_len, max_ctx,
                                         nb, bs, hq, hkv, d, _lib.dtype_code(q.dtype), _lib.ptr(buf), nbytes,
                                         _lib.stream_ptr(dev)), "tree_attention")
    return out


def accept_trees(tokens: torch.Tensor, targets: torch.Tensor, tree_mask: torch.Tensor, cu_q: torch.Tensor,
                 start_pos: torch.Tensor, max_q_len: int, k_cache: torch.Tensor | None = None,
                 v_cache: torch.Tensor | None = None, block_tables: torch.Tensor | None = None) -> Accepted:
    """The longest path of each request's tree that the model agrees with.

    tokens int64 (T,): the rows' token ids; targets int32 (T,): the model's
    next token after each row. The root is accepted; another node is when its
    ancestors are and its token is its parent's target. The deepest accepted
    node (the lowest of them) gives the path; the targets along it are the
    tokens the step yields. With the caches ((L, NB, bs, Hkv, D), or one
    layer's (NB, bs, Hkv, D)) and block_tables, the path's keys and values move
    in place to the positions start_pos, start_pos + 1, ..."""
    _lib.require_cuda(tokens, targets, tree_mask, cu_q, start_pos, k_cache, v_cache, block_tables)
    dev = tokens.device
    _int32("accept_trees", dev, targets, cu_q, start_pos)
    if tokens.dtype != torch.int64 or not tokens.is_contiguous():
        raise TypeError("accept_trees: tokens must be contiguous int64")
    T, B = tokens.numel(), start_pos.numel()
    if targets.numel() != T or cu_q.numel() != B + 1:
        raise ValueError("accept_trees: one target per token and one start position per request are needed")
    if B == 0:
        raise ValueError("accept_trees: empty batch")
    _mask_words("accept_trees", tree_mask, T, max_q_len, dev)
    L = nb = bs = hkv = d = width = code = 0
    if k_cache is not None or v_cache is not None:
        if k_cache is None or v_cache is None or block_tables is None:
            raise ValueError("accept_trees: the move needs both caches and block_tables")
        if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
            raise ValueError("accept_trees: K and V caches differ in shape or dtype")
        if not (k_cache.is_contiguous() and v_cache.is_contiguous()) or k_cache.device != dev or \
                v_cache.device != dev:
            raise ValueError("accept_trees: the caches must be contiguous and on the tokens' device")
        _int32("accept_trees", dev, block_tables)
        if block_tables.dim() != 2 or block_tables.shape[0] != B:
            raise ValueError("accept_trees: block_tables needs one row per request")
        if k_cache.dim() not in (4, 5):
            raise ValueError("accept_trees: caches are (L, NB, bs, Hkv, D) or one layer's (NB, bs, Hkv, D)")
        L = k_cache.shape[0] if k_cache.dim() == 5 else 1
        nb, bs, hkv, d = k_cache.shape[-4:]
        width = block_tables.shape[1]
        code = _lib.dtype_code(k_cache.dtype)
    num, start, nodes, out = torch.empty(2 * B + 2 * B * max_q_len, dtype=torch.int32, device=dev).split(
        [B, B, B * max_q_len, B * max_q_len])
    with torch.cuda.device(dev):
        _lib.check(_lib.load().ps_accept_trees(
            num.data_ptr(), nodes.data_ptr(), out.data_ptr(), start.data_ptr(), tokens.data_ptr(), targets.data_ptr(),
            tree_mask.data_ptr(), cu_q.data_ptr(), start_pos.data_ptr(), B, T, max_q_len, _lib.ptr(k_cache),
            _lib.ptr(v_cache), _lib.ptr(block_tables), width, L, nb, bs, hkv, d, code, _lib.stream_ptr(dev)),
            "accept_trees")
    return Accepted(num, nodes.view(B, max_q_len), out.view(B, max_q_len), start)
