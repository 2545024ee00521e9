"""Drafted-tree operators without a GPU: refusals of buffers that overlap,
shapes for tracing, scratch that captured calls go on using."""

import weakref

import pytest
import torch

from pageserve_b200 import _lib
from pageserve_b200.paged_attention import AttentionWorkspace
from pageserve_b200.quantization import LinearWorkspace

P = 1 << 20  # an aligned address that no check reads


def _lib_or_skip():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    return _lib.load()


# Ranges of a call that is in order: 3 requests, 40 rows in trees of up to 130, tables of 7, 9 free blocks.
IN = dict(tin=P + 0x1000, held=P + 0x2000, seq=P + 0x3000, q=P + 0x4000, free=P + 0x5000, par=P + 0x6000)
SIZE = dict(tables=3 * 7 * 4, held_out=12, cu=16, pos=160, slots=160, mask=40 * 3 * 8, used=4,
            tin=3 * 7 * 4, held=12, seq=12, q=12, free=36, par=160)


def _tables(lib, nb=64, **kw):
    a = dict(tables=P + 0x10000, held_out=P + 0x11000, cu=P + 0x12000, pos=P + 0x13000, slots=P + 0x14000,
             mask=P + 0x15000, used=P + 0x16000, **IN, B=3, T=40, max_q=130, width=7, nfree=9, nb=nb, bs=16)
    a.update(kw)
    return lib.ps_build_step_tables(*a.values(), None)


@pytest.mark.parametrize("out", ["tables", "held_out", "cu", "pos", "slots", "mask", "used"])
@pytest.mark.parametrize("src", list(IN))
def test_build_step_tables_refuses_outputs_over_inputs(out, src):
    """CTAs write a request's outputs while others still read every request's
    lengths, old entries and the free list. Both ends of the overlap."""
    lib = _lib_or_skip()
    for at in (IN[src] + SIZE[src] - 4, IN[src] - SIZE[out] + 4):
        assert _tables(lib, **{out: at}) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()


def test_build_step_tables_refuses_shifted_tables():
    """In place is the same address; one row further is not."""
    lib = _lib_or_skip()
    for shift in (-56, -28, 28, 56, 4):
        assert _tables(lib, tables=IN["tin"] + shift) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()


ACC_IN = dict(tok=P + 0x1000, tgt=P + 0x2000, mask=P + 0x3000, cu=P + 0x4000, sp=P + 0x5000, tab=P + 0x6000)
ACC_SIZE = dict(num=12, nodes=3 * 70 * 4, out=3 * 70 * 4, start_out=12, tok=320, tgt=160, mask=40 * 16, cu=16, sp=12,
                tab=3 * 8 * 4)


def _accept(lib, **kw):
    a = dict(num=P + 0x10000, nodes=P + 0x11000, out=P + 0x12000, start_out=P + 0x13000, tok=0, tgt=0, mask=0, cu=0,
             sp=0, B=3, T=40, max_q=70, k=P + 0x100000, v=P + 0x200000, tab=0, width=8, L=2, nb=16, bs=16, hkv=2, d=64,
             dt=_lib.PS_BF16)
    a.update(ACC_IN)
    a.update(kw)
    return lib.ps_accept_trees(*a.values(), None)


@pytest.mark.parametrize("out", ["num", "nodes", "out", "start_out"])
@pytest.mark.parametrize("src", list(ACC_IN))
def test_accept_trees_refuses_outputs_over_inputs(out, src):
    """One block of a request writes what the others still read."""
    lib = _lib_or_skip()
    for at in (ACC_IN[src] + ACC_SIZE[src] - 4, ACC_IN[src] - ACC_SIZE[out] + 4):
        assert _accept(lib, **{out: at}) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()


ATT_IN = dict(q=P + 0x10000, k=P + 0x40000, v=P + 0x80000, tab=P + 0x1000, cu=P + 0x2000, sp=P + 0x3000, mask=P + 0x4000)
ATT_SIZE = dict(q=8 * 4 * 128 * 2, k=16 * 16 * 2 * 128 * 2, v=16 * 16 * 2 * 128 * 2, tab=2 * 8 * 4, cu=12, sp=8,
                mask=64, out=8 * 4 * 128 * 2)


def _attn(lib, **kw):
    a = dict(out=P + 0x20000, **ATT_IN, B=2, T=8, max_q=4, max_ctx=100, nb=16, bs=16, hq=4, hkv=2, d=128,
             dt=_lib.PS_BF16, ws=P + 0x1000000, wsb=1 << 24)
    a = {k: a[k] for k in ("out", "q", "k", "v", "tab")} | {"width": 8} | {k: a[k] for k in list(a) if k not in (
        "out", "q", "k", "v", "tab")}
    a.update(kw)
    return lib.ps_tree_attention(*a.values(), None)


@pytest.mark.parametrize("src", list(ATT_IN))
def test_tree_attention_refuses_outputs_over_inputs(src):
    """Blocks finish at any time: what one writes another may still have to read."""
    lib = _lib_or_skip()
    last = (ATT_IN[src] + ATT_SIZE[src] - 1) // 16 * 16
    for at in (last, last - ATT_SIZE["out"] + 16):
        assert _attn(lib, out=at) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()
    for at in (last, last - 4096):
        assert _attn(lib, ws=at) == _lib.PS_ERR_INVALID
        assert "overlap" in _lib.last_error()
    assert _attn(lib, ws=P + 0x20000 + 16) == _lib.PS_ERR_INVALID and "overlap" in _lib.last_error()


@pytest.mark.parametrize("kind", [AttentionWorkspace, LinearWorkspace])
def test_workspace_keeps_what_a_graph_was_captured_with(kind, monkeypatch):
    """A captured graph holds the scratch's address, not the tensor: a later,
    larger call must not free it. What no graph was captured with is freed."""
    capturing = False
    monkeypatch.setattr(kind, "_capturing", staticmethod(lambda buf: capturing))
    ws = kind()
    first = weakref.ref(ws.get(1000, "cpu"))
    capturing = True
    assert ws.get(500, "cpu") is first() and ws.get(0, "cpu") is None
    capturing = False
    second = weakref.ref(ws.get(1001, "cpu"))
    assert second() is not first() and second().numel() == 1001
    third = weakref.ref(ws.get(1002, "cpu"))
    assert first() is not None and second() is None and ws.get(7, "cpu") is third()


def test_workspace_of_several_devices():
    """A call on another device neither frees nor grows what the first one has."""
    ws = AttentionWorkspace()
    a, b = ws.get(1000, "cpu"), ws.get(600, "meta")
    for _ in range(50):
        assert ws.get(1000, torch.device("cpu")) is a and ws.get(600, torch.device("meta")) is b


def test_out_forms_have_meta_functions():
    """Fake-tensor tracing of the forms that write into a given tensor (the
    model's step calls one)."""
    from pageserve_b200 import ops as torch_ops
    if not torch_ops.LIB_PATH.exists():
        pytest.skip("libpageserve_torch_ops.so is not built")
    ns = torch_ops.load()
    i = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")  # noqa: E731
    r = ns.build_step_tables_out(i(3, 7), i(3), i(3), i(3, 7), i(3), i(9), 9, 16, 20, i(20), 70)
    assert [tuple(x.shape) for x in r] == [(3,), (4,), (20,), (20,), (20, 2), (1,)]
    assert [x.dtype for x in r] == [torch.int32] * 4 + [torch.int64, torch.int32]
    r = ns.build_step_tables_out(i(3, 7), i(3), i(3), i(3, 7), i(3), i(9), 9, 16, 20)
    assert r[4].shape == (0,)
    q = torch.empty(20, 4, 64, dtype=torch.bfloat16, device="meta")
    kv = torch.empty(9, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    mask = torch.empty(20, 2, dtype=torch.int64, device="meta")
    assert ns.tree_attention_out(torch.empty_like(q), q, kv, kv, i(3, 7), i(4), i(3), mask, 70, 112) is None


def test_every_operator_has_a_meta_function():
    from pageserve_b200 import ops as torch_ops
    if not torch_ops.LIB_PATH.exists():
        pytest.skip("libpageserve_torch_ops.so is not built")
    torch_ops.load()
    for name in ("build_step_tables", "build_step_tables_out", "tree_attention", "tree_attention_out", "accept_trees"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"pageserve_b200::{name}", "Meta"), name
