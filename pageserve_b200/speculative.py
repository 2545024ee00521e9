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
lengths stay on the device, so a step can be captured in a CUDA graph (after one
call outside it).
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


_ops = None


def _op(name: str):
    """The torch operator (torch_ops/pageserve_ops.cpp: the argument checks,
    the output allocations and the C call of each function below)."""
    global _ops
    if _ops is None:
        from . import ops
        ns = ops.load()
        _ops = {n: getattr(ns, n).default for n in ("build_step_tables", "build_step_tables_out", "tree_attention",
                                                    "tree_attention_out", "accept_trees")}
    return _ops[name]


def build_step_tables(seq_lens: torch.Tensor, q_lens: torch.Tensor, block_tables: torch.Tensor, held: torch.Tensor,
                      free_blocks: torch.Tensor, num_blocks: int, block_size: int, total_tokens: int,
                      parents: torch.Tensor | None = None, max_q_len: int | None = None,
                      out: torch.Tensor | None = None, max_ctx: int | None = None) -> StepTables:
    """Block tables, positions, slots and ancestor masks of one step.

    seq_lens, q_lens, held int32 (B,): each request's cached tokens, new tokens
    (0: it waits) and blocks in its row of block_tables int32 (B, max_blocks).
    Missing blocks are taken from free_blocks int32 (F,) in request order.
    total_tokens: the step's rows (at least the sum of q_lens; the rows behind
    get position 0, slot -1). parents int32 (total_tokens,): each row's parent
    among its request's rows, -1 for none; a row's position is then its depth
    past seq_len, and tree_mask is made (max_q_len bounds q_lens, at most
    256). Without parents the rows are a chunk at seq_len + i. ``out`` takes
    the tables; it may be block_tables itself, but must not overlap it or another
    input in any other way. A free list that is too short
    leaves -1 entries and slots, free_used above F and device error 6; lengths
    beyond the given bounds are device error 5 (``_lib.raise_on_device_error``).
    In a tree the rows from the first one without a slot on get mask 0, as do
    all rows of a request whose context passes its table row or ``max_ctx``
    (give the bound that :func:`tree_attention` gets), so that
    :func:`accept_trees` keeps nothing that is not in the cache or that the
    attention leaves out."""
    _lib.require_cuda(seq_lens)
    if out is None:
        r = _op("build_step_tables")(seq_lens, q_lens, block_tables, held, free_blocks, num_blocks, block_size,
                                     total_tokens, parents, max_q_len, max_ctx)
    else:
        r = (out, *_op("build_step_tables_out")(out, seq_lens, q_lens, block_tables, held, free_blocks, num_blocks,
                                                block_size, total_tokens, parents, max_q_len, max_ctx))
    if parents is None:
        r = (*r[:5], None, r[6])
    return StepTables._make(r)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                   cu_q: torch.Tensor, start_pos: torch.Tensor, tree_mask: torch.Tensor, max_q_len: int, max_ctx: int,
                   out: torch.Tensor | None = None, workspace: AttentionWorkspace | None = None) -> torch.Tensor:
    """Paged attention of drafted trees: q (total_q, Hq, D), caches (NB, bs,
    Hkv, D), tables, cu_q and start_pos as in ``paged_attention``; tree_mask
    int64 (total_q, ceil(max_q_len / 64)) from :func:`build_step_tables`.
    Node i of request b sees the cached keys [0, start_pos[b]) and the nodes
    of its mask row (stored at start_pos[b] + node); 0 when it sees nothing.
    Rows of ``out`` (which must not overlap an input) behind cu_q[-1] are left
    as they were. A workspace serves calls on one stream at a time; without one
    the scratch is allocated per call."""
    _lib.require_cuda(q)
    buf = None
    if workspace is not None:
        B, (_, hq, d), hkv = start_pos.numel(), q.shape, k_cache.shape[-2]
        nbytes = _lib.load().ps_tree_attention_workspace_size(B, max_q_len, max_ctx, hq, hkv, d)
        buf = workspace.get(nbytes, q.device)
    if out is None:
        return _op("tree_attention")(q, k_cache, v_cache, block_tables, cu_q, start_pos, tree_mask, max_q_len, max_ctx,
                                     buf)
    _op("tree_attention_out")(out, q, k_cache, v_cache, block_tables, cu_q, start_pos, tree_mask, max_q_len, max_ctx,
                              buf)
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
    in place to the positions start_pos, start_pos + 1, ... A node that the
    table has no block for is a device error (1, 5), and ``start_pos`` of the
    result ends before it: only what precedes it is in the cache."""
    _lib.require_cuda(tokens)
    return Accepted._make(_op("accept_trees")(tokens, targets, tree_mask, cu_q, start_pos, max_q_len, k_cache, v_cache,
                                              block_tables))
