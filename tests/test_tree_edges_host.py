"""Drafted-tree operators without a GPU: refusals of buffers that overlap,
shapes for tracing, scratch that captured calls go on using."""

import pytest

from pageserve_b200 import _lib

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
