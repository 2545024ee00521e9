"""Drafted-tree operators where a step cannot be carried out in full, where
cached values are not finite, and how far results may be off on average."""

import numpy as np
import pytest
import torch

from oracle import tree
from test_gpu_speculative import _case, _run, _status, dev  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------- values that are not finite --

def _with_value(c, dev, places, heads):
    """The case's result with V[key, kv head 0, column 3] of request 0 set, and
    the same without it; everything else must be the same bits."""
    clean = _run(c, dev).double().cpu()
    for key, value in places:
        c["v"][c["tab"][0, key // c["bs"]], key % c["bs"], 0, 3] = value
    got = _run(c, dev).double().cpu()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:c["cu"][1], :heads, 3] = False
    assert torch.equal(got[rest], clean[rest])
    return got[:c["cu"][1], :heads, 3]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("ctx,key", [(61, 60), (61, 0), (700, 5), (700, 639), (700, 699), (3000, 1300)])
@pytest.mark.parametrize("D,bs,nodes,bound", [(128, 16, 6, 6), (64, 16, 6, 6), (128, 16, 6, 40), (64, 16, 20, 20),
                                              (128, 4, 6, 6), (64, 4, 20, 40), (128, 16, 70, 70)])
def test_attention_cached_values_that_are_not_finite(dev, value, ctx, key, D, bs, nodes, bound):  # noqa: F811
    """A cached V value that is not finite reaches every row with its weight:
    infinity stays infinity, whatever bound the call gives for its rows."""
    c = _case(40, [ctx, 40], [nodes, 5], 8, 2, D, bs, torch.float16 if D == 64 else torch.bfloat16)
    c["max_q"] = max(bound, c["max_q"])
    col = _with_value(c, dev, [(key, value)], 4)
    assert torch.isnan(col).all() if value != value else (col == value).all()
    assert _status() == 0


@pytest.mark.parametrize("D,bs,nodes", [(128, 16, 6), (64, 16, 20), (128, 4, 6)])
def test_attention_cached_infinities_of_both_signs(dev, D, bs, nodes):  # noqa: F811
    c = _case(41, [900, 40], [nodes, 5], 8, 2, D, bs, torch.bfloat16)
    col = _with_value(c, dev, [(100, float("inf")), (200, float("inf"))], 4)
    assert (col == float("inf")).all()
    col = _with_value(_case(41, [900, 40], [nodes, 5], 8, 2, D, bs, torch.bfloat16), dev,
                      [(100, float("inf")), (800, float("-inf"))], 4)
    assert torch.isnan(col).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,bs,nodes,ctx", [(128, 16, 6, 700), (64, 16, 20, 700), (128, 4, 6, 700), (128, 16, 6, 6000),
                                            (128, 4, 20, 6000)])
def test_attention_infinity_of_small_weight(dev, D, bs, nodes, ctx, dtype):  # noqa: F811
    """Weights of cached infinities of e^-360, far below the 16-bit types and
    32-bit floats, beside keys that hold the maximum: in one tile, in another
    of the same share, and in another share, whose other keys weigh e^-120."""
    for key in (3, 130, ctx // 2, ctx - 1):
        c = _case(42, [ctx, 40], [nodes, 5], 8, 2, D, bs, dtype)
        n = ctx + nodes
        blk = torch.as_tensor(c["tab"][0][np.arange(n) // bs])
        off = torch.as_tensor(np.arange(n) % bs)
        # all queries share a direction: its score is 0 except at two keys, where it is large, and at `key`
        c["q"][:] = (c["q"].float() * 0.1).to(dtype)
        c["q"][..., 0] = 8.0
        c["k"][blk, off] = (c["k"][blk, off].float() * 0.1).to(dtype)
        c["k"][blk, off, :, 0] = 0.0
        for at in (50, ctx // 3):
            c["k"][blk[at], off[at], :, 0] = 15.0 * D ** 0.5
        c["k"][blk[key], off[key], :, 0] = -30.0 * D ** 0.5  # 45 x 8 = 360 below the largest
        col = _with_value(c, dev, [(key, float("inf"))], 4)
        assert (col == float("inf")).all(), key
    assert _status() == 0
