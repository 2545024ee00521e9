"""Drafted-tree operators without a GPU: the 64-bit oracle on worked examples,
and the entry points' refusals (all of them before any launch)."""

import numpy as np
import pytest
import torch

from oracle import tree
from pageserve_b200 import _lib


def test_oracle_tables_worked_example():
    # block size 4; request 0 has 6 cached tokens in 2 blocks and 3 new ones (a fork), request 1 is new
    tab, held, cu, pos, slots, mask, used = tree.step_tables(
        [6, 0], [3, 5], [[9, 2, -1], [-1, -1, -1]], [2, 0], [7, 5, 1], 4, 10, parents=[-1, 0, 0, -1, 0, 1, 1, 3, -1, -1],
        max_q_len=5)
    assert tab.tolist() == [[9, 2, 7], [5, 1, -1]] and held.tolist() == [3, 2] and used == 3
    assert cu.tolist() == [0, 3, 8]
    assert slots.tolist() == [2 * 4 + 2, 2 * 4 + 3, 7 * 4, 5 * 4, 5 * 4 + 1, 5 * 4 + 2, 5 * 4 + 3, 1 * 4, -1, -1]
    assert pos.tolist() == [6, 7, 7, 0, 1, 2, 2, 3, 0, 0]
    assert mask[:, 0].tolist() == [1, 3, 5, 1, 3, 7, 11, 27, 0, 0]


def test_oracle_attention_is_causal_attention_on_a_chain():
    from oracle import ops
    rng = np.random.default_rng(0)
    q = rng.standard_normal((5, 4, 8)).astype(np.float32)
    kc = rng.standard_normal((6, 4, 2, 8)).astype(np.float32)
    vc = rng.standard_normal((6, 4, 2, 8)).astype(np.float32)
    sets = tree.ancestors([-1, 0, 1, 2, 3])
    out, _ = tree.tree_attention(q, kc, vc, [[4, 1, 0, 3]], [0, 5], [7], sets)
    ref = ops.paged_causal_attention_incremental(q, kc, vc, [4, 1, 0, 3], 4, 7)
    assert np.abs(out - ref).max() < 1e-5


def test_oracle_acceptance_worked_example():
    #      0 -> 1 -> 3, 0 -> 2 -> 4 -> 5; the model agrees with 2 and 4, not with 5
    sets = tree.ancestors([-1, 0, 0, 1, 2, 4])
    assert tree.accept([10, 11, 12, 13, 14, 15], [12, 13, 14, 99, 98, 97], sets) == [0, 2, 4]
    assert tree.accept([10, 11, 12, 13, 14, 15], [1, 1, 1, 1, 1, 1], sets) == [0]
    cache = np.arange(6, dtype=np.float64).reshape(1, 3, 2, 1, 1).copy()
    tree.move_rows(cache, [0, 1, 2], 2, 0, [0, 2, 4])
    assert cache.reshape(-1).tolist() == [0, 2, 4, 3, 4, 5]


def _lib_or_skip():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    return _lib.load()


P = 1 << 20  # an aligned address that no check reads


def _tables(lib, **kw):
    a = dict(tables=P, held_out=P, cu=P, pos=P, slots=P, mask=P, used=P, tin=P, held=2 * P, seq=P + 64, q=P + 128, free=P,
             par=P, B=2, T=8, max_q=4, width=4, nfree=4, nb=16, bs=16)
    a.update(kw)
    return lib.ps_build_step_tables(*a.values(), None)


def test_build_step_tables_refusals():
    lib = _lib_or_skip()
    assert _tables(lib, B=0) == _lib.PS_ERR_INVALID
    assert _tables(lib, bs=0) == _lib.PS_ERR_INVALID
    assert _tables(lib, T=-1) == _lib.PS_ERR_INVALID
    assert _tables(lib, mask=None) == _lib.PS_ERR_INVALID
    assert _tables(lib, seq=None) == _lib.PS_ERR_INVALID
    assert _tables(lib, free=None) == _lib.PS_ERR_INVALID
    assert _tables(lib, held_out=2 * P) == _lib.PS_ERR_INVALID  # aliases held
    assert _tables(lib, max_q=0) == _lib.PS_ERR_INVALID
    assert _tables(lib, max_q=257) == _lib.PS_ERR_UNSUPPORTED
    assert _tables(lib, nb=1 << 28, bs=16) == _lib.PS_ERR_INVALID  # slots past 32 bits


def _attn(lib, **kw):
    a = dict(out=P, q=P, k=P, v=P, tab=P, width=8, cu=P, sp=P, mask=P, B=2, T=8, max_q=4, max_ctx=100, nb=16, bs=16,
             hq=4, hkv=2, d=128, dt=_lib.PS_BF16, ws=P, wsb=1 << 40)
    a.update(kw)
    return lib.ps_tree_attention(*a.values(), None)


def test_tree_attention_refusals():
    lib = _lib_or_skip()
    assert _attn(lib, B=0) == _lib.PS_ERR_INVALID
    assert _attn(lib, hq=5) == _lib.PS_ERR_INVALID
    assert _attn(lib, max_ctx=129) == _lib.PS_ERR_INDEX
    assert _attn(lib, max_ctx=3) == _lib.PS_ERR_INVALID  # below max_q_len
    assert _attn(lib, max_q=257, max_ctx=300, width=64) == _lib.PS_ERR_UNSUPPORTED
    assert _attn(lib, d=96) == _lib.PS_ERR_UNSUPPORTED
    assert _attn(lib, dt=_lib.PS_F32) == _lib.PS_ERR_UNSUPPORTED
    assert _attn(lib, mask=None) == _lib.PS_ERR_INVALID
    assert _attn(lib, q=P + 8) == _lib.PS_ERR_INVALID
    assert _attn(lib, ws=None) == _lib.PS_ERR_INVALID
    assert _attn(lib, wsb=16) == _lib.PS_ERR_INVALID
    assert "workspace" in _lib.last_error()
    assert _attn(lib, T=0) == _lib.PS_OK  # nothing to do, nothing launched
    assert lib.ps_tree_attention_workspace_size(2, 4, 100, 4, 2, 128) > 0
    assert lib.ps_tree_attention_workspace_size(2, 300, 400, 4, 2, 128) == 0
    # bounded whatever the context: partials of at most two row tiles per CTA
    assert lib.ps_tree_attention_workspace_size(128, 256, 1 << 20, 64, 8, 128) < 64 << 20


def _accept(lib, **kw):
    a = dict(num=P, nodes=P, out=P, start_out=P, tok=P, tgt=P, mask=P, cu=P + 64, sp=P + 128, B=2, T=8, max_q=4, k=P, v=P,
             tab=P, width=8, L=2, nb=16, bs=16, hkv=2, d=64, dt=_lib.PS_BF16)
    a.update(kw)
    return lib.ps_accept_trees(*a.values(), None)


def test_accept_trees_refusals():
    lib = _lib_or_skip()
    assert _accept(lib, B=0) == _lib.PS_ERR_INVALID
    assert _accept(lib, max_q=257) == _lib.PS_ERR_UNSUPPORTED
    assert _accept(lib, tgt=None) == _lib.PS_ERR_INVALID
    assert _accept(lib, start_out=P + 128) == _lib.PS_ERR_INVALID  # aliases start_pos
    assert _accept(lib, v=None) == _lib.PS_ERR_INVALID
    assert _accept(lib, tab=None) == _lib.PS_ERR_INVALID
    assert _accept(lib, dt=_lib.PS_I8) == _lib.PS_ERR_UNSUPPORTED
    assert _accept(lib, hkv=1, d=4) == _lib.PS_ERR_INVALID  # rows of 8 bytes
    assert _accept(lib, k=P + 8) == _lib.PS_ERR_INVALID


def test_cpu_tensors_raise():
    from pageserve_b200 import speculative as sp
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    m = torch.zeros(1, 1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        sp.build_step_tables(i, i, i.view(1, 1), i, i, 4, 16, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        sp.tree_attention(x, c, c, i.view(1, 1), i, i, m, 1, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        sp.accept_trees(m.view(-1), i, m, i, i, 1)


def test_torch_operators_have_meta_shapes():
    """Fake-tensor tracing sees each operator's outputs."""
    from pageserve_b200 import ops as torch_ops
    if not torch_ops.LIB_PATH.exists():
        pytest.skip("libpageserve_torch_ops.so is not built")
    ns = torch_ops.load()
    i = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")  # noqa: E731
    r = ns.build_step_tables(i(3), i(3), i(3, 7), i(3), i(9), 9, 16, 20, i(20), 70)
    assert [tuple(x.shape) for x in r] == [(3, 7), (3,), (4,), (20,), (20,), (20, 2), (1,)]
    assert [x.dtype for x in r] == [torch.int32] * 5 + [torch.int64, torch.int32]
    r = ns.build_step_tables(i(3), i(3), i(3, 7), i(3), i(9), 9, 16, 20)
    assert r[5].shape == (0,)
    q = torch.empty(20, 4, 64, dtype=torch.bfloat16, device="meta")
    kv = torch.empty(9, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    mask = torch.empty(20, 2, dtype=torch.int64, device="meta")
    out = ns.tree_attention(q, kv, kv, i(3, 7), i(4), i(3), mask, 70, 112)
    assert out.shape == q.shape and out.dtype == q.dtype
    tok = torch.empty(20, dtype=torch.int64, device="meta")
    r = ns.accept_trees(tok, i(20), mask, i(4), i(3), 70)
    assert [tuple(x.shape) for x in r] == [(3,), (3, 70), (3, 70), (3,)] and all(x.dtype == torch.int32 for x in r)


def test_accept_trees_refuses_overlapping_caches():
    """K and V rows move at the same time: one cache as both, or two that
    overlap, would lose rows."""
    lib = _lib_or_skip()
    size = 2 * 16 * 16 * 2 * 64 * 2  # bytes of a cache of _accept's sizes
    for v in (P, P + 16, P + size - 16):
        assert _accept(lib, v=v) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()
        assert _accept(lib, k=v, v=P) == _lib.PS_ERR_INVALID
