"""Drafted-tree operators on the GPU against the 64-bit oracle."""

import numpy as np
import pytest
import torch

from oracle import tree

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from pageserve_b200 import _lib
    _lib.load()
    d = torch.device("cuda", 0)
    _lib.ensure_status_word(d)
    _lib.device_status(clear=True)
    return d


def _status():
    from pageserve_b200 import _lib
    return _lib.device_status(clear=True)


def _i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(dev)


def _parents(rng, n, kind="random"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)]


# -------------------------------------------------------- build_step_tables --

def _check_tables(dev, seq, q, bs, width, total=None, parents=None, held=None, seed=0, inplace=False):
    from pageserve_b200 import speculative as sp
    rng = np.random.default_rng(seed)
    B = len(seq)
    held = [(s + bs - 1) // bs for s in seq] if held is None else held
    need = [max(h, (s + n + bs - 1) // bs) for h, s, n in zip(held, seq, q)]
    nb = sum(need) + 5
    perm = rng.permutation(nb)
    tab = np.full((B, width), -1, np.int64)
    at = 0
    for b, h in enumerate(held):
        tab[b, :h] = perm[at:at + h]
        at += h
    free = perm[at:]
    total = sum(q) if total is None else total
    mq = max(1, max(q))
    ref = tree.step_tables(seq, q, tab, held, free, bs, total, parents, mq)
    t = _i32(tab, dev)
    r = sp.build_step_tables(_i32(seq, dev), _i32(q, dev), t, _i32(held, dev), _i32(free, dev), nb, bs, total,
                             parents=None if parents is None else _i32(parents, dev), max_q_len=mq,
                             out=t if inplace else None)
    assert _status() == 0
    assert (r.block_tables is t) == inplace
    assert r.block_tables.cpu().tolist() == ref[0].tolist()
    assert r.held.cpu().tolist() == ref[1].tolist()
    assert r.cu_q.cpu().tolist() == ref[2].tolist()
    assert r.positions.cpu().tolist() == ref[3].tolist()
    assert r.slots.cpu().tolist() == ref[4].tolist()
    if parents is None:
        assert r.tree_mask is None
    else:
        assert np.array_equal(r.tree_mask.cpu().numpy(), ref[5])
    assert int(r.free_used) == ref[6]


@pytest.mark.parametrize("bs", [1, 3, 16, 64])
@pytest.mark.parametrize("B", [1, 2, 31, 300, 777])
def test_tables_of_chunks(dev, B, bs):
    rng = np.random.default_rng(B * 100 + bs)
    seq = rng.integers(0, 200, B).tolist()
    q = rng.integers(0, 4, B).tolist()
    q[B // 2] = 300  # a prompt chunk longer than a CTA
    _check_tables(dev, seq, q, bs, width=(500 + bs - 1) // bs + 2, total=sum(q) + 5)
    _check_tables(dev, seq, q, bs, width=(500 + bs - 1) // bs, held=[0] * B, inplace=True)


def test_tables_of_empty_and_full_rows(dev):
    _check_tables(dev, [0], [0], 16, 1, total=0)
    _check_tables(dev, [0, 0, 0], [0, 0, 0], 16, 4, total=2)
    _check_tables(dev, [15, 16, 17, 32], [1, 1, 1, 0], 16, 2, total=3)
    _check_tables(dev, [5, 5], [1, 1], 16, 4, held=[3, 1])  # blocks held ahead stay


@pytest.mark.parametrize("kind", ["random", "chain", "star"])
@pytest.mark.parametrize("n", [1, 2, 33, 64, 65, 130, 256])
def test_tables_of_trees(dev, n, kind):
    rng = np.random.default_rng(n)
    q = [n, 0, max(1, n // 3), n]
    par = sum((_parents(rng, x, kind) for x in q if x), [])
    _check_tables(dev, [31, 9, 0, 2048], q, 16, 160, total=len(par) + 2, parents=par + [-1, -1], seed=n)


def test_tables_forest_and_bad_parents(dev):
    from pageserve_b200 import speculative as sp
    _check_tables(dev, [4], [5], 4, 4, parents=[-1, -1, 0, 1, -1])
    r = sp.build_step_tables(_i32([4], dev), _i32([4], dev), _i32([[3, 1, 2]], dev), _i32([3], dev), _i32([0], dev), 8, 4,
                             4, parents=_i32([-1, 1, 9, -7], dev), max_q_len=4)
    assert _status() == 5  # parents outside [-1, i) count as none
    assert r.tree_mask.cpu().tolist() == [[1], [2], [4], [8]]
    assert r.positions.cpu().tolist() == [4, 4, 4, 4]


def test_tables_short_free_list(dev):
    from pageserve_b200 import speculative as sp
    r = sp.build_step_tables(_i32([0, 8], dev), _i32([9, 9], dev), _i32([[-1] * 5, [5, 6, -1, -1, -1]], dev),
                             _i32([0, 2], dev), _i32([7, 1, 2, 3], dev), 8, 4, 18)
    assert _status() == 6
    assert int(r.free_used) == 6
    assert r.block_tables.cpu().tolist() == [[7, 1, 2, -1, -1], [5, 6, 3, -1, -1]]
    assert r.held.cpu().tolist() == [3, 3]
    s = r.slots.cpu().tolist()
    assert s[:9] == [28, 29, 30, 31, 4, 5, 6, 7, 8]
    assert s[9:] == [12, 13, 14, 15] + [-1] * 5


def test_tables_bounds_are_recorded(dev):
    from pageserve_b200 import speculative as sp

    def run(seq, q, held, total, par=None, mq=None, tab=((0, 1),)):
        r = sp.build_step_tables(_i32(seq, dev), _i32(q, dev), _i32(tab, dev), _i32(held, dev), _i32([2, 3], dev), 4, 4,
                                 total, parents=None if par is None else _i32(par, dev), max_q_len=mq)
        return r, _status()

    r, e = run([-3], [2], [1], 2)
    assert e == 5 and r.positions.cpu().tolist() == [0, 1]
    r, e = run([7], [4], [2], 4)  # context 11 past a table of 2 x 4
    assert e == 5 and r.slots.cpu().tolist() == [7, -1, -1, -1] and r.held.cpu().tolist() == [2]
    r, e = run([0], [6], [0], 4)  # more rows than the step has
    assert e == 5 and r.cu_q.cpu().tolist() == [0, 4]
    r, e = run([0], [3], [0], 3, par=[-1, 0, 1], mq=2)  # more nodes than max_q_len
    assert e == 5 and r.tree_mask.cpu().tolist() == [[1], [3], [0]] and r.slots.cpu().tolist() == [8, 9, -1]
    r, e = run([1], [1], [1], 1, tab=((9, 1),))  # a held block outside the pool
    assert e == 1 and r.slots.cpu().tolist() == [-1]
    r, e = run([2 ** 31 - 2], [3], [0], 3)  # sums past 32 bits
    assert e == 5 and r.slots.cpu().tolist() == [-1, -1, -1]


def test_tables_python_refusals(dev):
    from pageserve_b200 import speculative as sp
    i = _i32([1], dev)
    t = _i32([[0, 1]], dev)
    with pytest.raises(TypeError):
        sp.build_step_tables(i.long(), i, t, i, i, 4, 4, 1)
    with pytest.raises(ValueError):
        sp.build_step_tables(i, _i32([1, 1], dev), t, i, i, 4, 4, 1)
    with pytest.raises(ValueError):
        sp.build_step_tables(i, i, t, i, i, 4, 4, 2, parents=i, max_q_len=1)
    with pytest.raises(ValueError):
        sp.build_step_tables(i, i, t, i, i, 4, 4, 1, parents=i)
    with pytest.raises(NotImplementedError):
        sp.build_step_tables(i, i, t, i, i, 4, 4, 1, parents=i, max_q_len=257)
    with pytest.raises(ValueError):
        sp.build_step_tables(i, i, t, i, i, 4, 4, 1, out=_i32([[0]], dev))


# ------------------------------------------------------------ tree_attention --

def _case(seed, ctxs, nodes, Hq, Hkv, D, bs, dtype, kind="random", stale=0.0):
    """CPU inputs rounded to dtype (as float64 arrays) and their tensors."""
    rng = np.random.default_rng(seed)
    B = len(ctxs)
    need = [(c + n + bs - 1) // bs for c, n in zip(ctxs, nodes)]
    nb = sum(need) + 3
    perm = rng.permutation(nb)
    width = max(need) + 1
    tab = np.full((B, width), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        tab[b, :n] = perm[at:at + n]
        at += n
    T = sum(nodes)
    q = torch.from_numpy(rng.standard_normal((T, Hq, D), dtype=np.float32)).to(dtype)
    k = torch.from_numpy(rng.standard_normal((nb, bs, Hkv, D), dtype=np.float32)).to(dtype)
    v = torch.from_numpy(rng.standard_normal((nb, bs, Hkv, D), dtype=np.float32)).to(dtype)
    if stale:  # whatever the context does not cover
        used = np.zeros((nb, bs), bool)
        for b in range(B):
            for p in range(ctxs[b] + nodes[b]):
                used[tab[b, p // bs], p % bs] = True
        k[torch.from_numpy(~used)] = stale
        v[torch.from_numpy(~used)] = stale
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(int)
    sets = []
    for n in nodes:
        sets += tree.ancestors(_parents(rng, n, kind)) if n else []
    return dict(q=q, k=k, v=v, tab=tab, cu=cu, sp=list(ctxs), sets=sets, max_q=max(1, max(nodes)), bs=bs,
                max_ctx=max(max(1, c + n) for c, n in zip(ctxs, nodes)))


def _run(c, dev, **kw):
    from pageserve_b200 import speculative as sp
    mask = torch.from_numpy(tree.mask_words(c["sets"], (c["max_q"] + 63) // 64)).to(dev)
    return sp.tree_attention(c["q"].to(dev), c["k"].to(dev), c["v"].to(dev), _i32(c["tab"], dev), _i32(c["cu"], dev),
                             _i32(c["sp"], dev), mask, c["max_q"], max(c["max_ctx"], c["max_q"]), **kw)


def _tolerance(c, ref, mag):
    """What the arithmetic may be off by. u: half a step of the type. The
    output's rounding u |o|; each weight's rounding u (its term of the sum of
    w |v|) and, for f16 weights below 2^-14, half a subnormal step 2^-25; they
    are powers 2^(s - r) with r the largest score rounded up to a whole number
    (or a lower one), so the largest weight and with it the sum is at least
    1/2, and the step counts 2^-24 after the division; scores in 32 bits, D products whose magnitudes
    sum to at most |q| |k|, each sum off by 2^-23 of it (the accumulator may
    truncate): a relative error of twice that in a weight, twice for weight and
    sum; the exponential and the join, 2^-20; sums over n keys, n 2^-23."""
    dt = c["q"].dtype
    u = torch.finfo(dt).eps / 2
    D = c["q"].shape[-1]
    qn = float(c["q"].double().norm(dim=-1).max())
    k = c["k"].double()
    kn = float(k.norm(dim=-1).nan_to_num(0, 0, 0).max())
    n = c["max_ctx"]
    delta = D * 2.0 ** -23 * qn * kn / np.sqrt(D)
    vmax = float(c["v"].double().abs().nan_to_num(0, 0, 0).max())
    sub = n * 2.0 ** -24 * vmax if dt == torch.float16 else 0.0
    return u * np.abs(ref) + (u + 4 * delta + 2.0 ** -20 + n * 2.0 ** -23) * 1.01 * mag + sub + 1e-30


def _check(c, dev, **kw):
    out = _run(c, dev, **kw).double().cpu().numpy()
    assert _status() == 0
    ref, mag = tree.tree_attention(c["q"].double().numpy(), c["k"].double().numpy(), c["v"].double().numpy(), c["tab"],
                                   c["cu"], c["sp"], c["sets"])
    err = np.abs(out - ref)
    tol = _tolerance(c, ref, mag)
    assert np.isfinite(out).all()
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (worst, err[worst], tol[worst], out[worst], ref[worst])


HEADS = [(14, 2, 64), (16, 2, 128), (40, 8, 128), (4, 4, 64), (3, 1, 128), (32, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("ctxs,nodes", [
    ([0], [1]), ([1], [1]), ([0, 0], [5, 1]), ([37], [7]), ([63, 64, 65], [1, 2, 3]), ([127, 128, 129, 0], [16, 1, 0, 16]),
    ([300, 5, 511], [33, 64, 1])])
def test_attention_small(dev, ctxs, nodes, Hq, Hkv, D, dtype):
    _check(_case(1, ctxs, nodes, Hq, Hkv, D, 16, dtype), dev)


@pytest.mark.parametrize("bs", [1, 4, 8, 16, 24, 32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 64), (16, 2, 128)])
def test_attention_block_sizes(dev, bs, Hq, Hkv, D):
    _check(_case(2, [250, 383, 3], [9, 20, 13], Hq, Hkv, D, bs, torch.bfloat16), dev)


@pytest.mark.parametrize("n", [1, 17, 63, 64, 65, 128, 129, 200, 256])
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_attention_tree_sizes(dev, n, kind):
    _check(_case(n, [100, 70], [n, (n + 1) // 2], 8, 2, 64, 16, torch.float16, kind), dev)


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(16, 2, 128, torch.bfloat16), (14, 2, 64, torch.float16)])
def test_attention_split_contexts(dev, Hq, Hkv, D, dtype):
    """Long contexts that several CTAs share, next to short ones."""
    _check(_case(3, [5000, 1, 2048, 700], [3, 1, 8, 11], Hq, Hkv, D, 16, dtype), dev)


def test_attention_many_requests(dev):
    rng = np.random.default_rng(5)
    ctxs, nodes = rng.integers(0, 60, 300).tolist(), rng.integers(0, 5, 300).tolist()
    _check(_case(4, ctxs, nodes, 4, 2, 64, 16, torch.bfloat16), dev)


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 16), (64, 4), (128, 64)])
def test_attention_stale_slots(dev, stale, D, bs):
    """Slots that no context covers hold anything."""
    _check(_case(6, [29, 100, 0, 1000], [6, 1, 3, 70], 8, 2, D, bs, torch.bfloat16, stale=stale), dev)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D,bs,ctx", [(128, 16, 61), (64, 16, 700), (128, 4, 61), (128, 16, 3000)])
def test_attention_node_with_values_that_are_not_finite(dev, value, D, bs, ctx):
    """A drafted node whose K and V overflowed reaches the nodes that see it
    and no other."""
    c = _case(7, [ctx, 40], [20, 5], 8, 2, D, bs, torch.float16)
    clean = _run(c, dev).double().cpu()
    node = 7
    pos = ctx + node
    sees = torch.tensor([node in s for s in c["sets"][:20]] + [False] * 5)
    v0 = c["v"].clone()
    blk, off = c["tab"][0, pos // bs], pos % bs
    c["v"][blk, off, 0, 3] = value
    got = _run(c, dev).double().cpu()
    assert torch.equal(got[~sees], clean[~sees])
    want = clean.clone()
    want[:, :4, 3] = torch.where(sees[:, None], torch.tensor(value, dtype=torch.float64), clean[:, :4, 3])
    if value != value:
        assert torch.isnan(got[sees][:, :4, 3]).all()
    else:
        assert torch.equal(got[:, :4, 3], want[:, :4, 3])
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:, :4, 3] = False
    assert torch.equal(got[rest], clean[rest])
    c["v"] = v0
    c["k"][blk, off, 1] = value  # a masked score that is not finite
    got = _run(c, dev).double().cpu()
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.equal(got[:, :4], clean[:, :4])
    assert _status() == 0


def test_attention_rows_that_see_nothing(dev):
    c = _case(8, [0, 50], [4, 3], 8, 2, 128, 16, torch.bfloat16)
    c["sets"][2] = set()
    c["sets"][5] = set()  # sees its context alone
    _check(c, dev)
    assert (_run(c, dev)[2] == 0).all()


def test_attention_nodes_need_not_see_themselves(dev):
    """Masks are the caller's: any set of the request's nodes."""
    rng = np.random.default_rng(9)
    c = _case(9, [30, 0], [90, 66], 4, 2, 64, 16, torch.bfloat16)
    c["sets"] = [set(np.nonzero(rng.random(n) < 0.3)[0].tolist()) for n in [90] * 90 + [66] * 66]
    _check(c, dev)


def test_attention_leaves_rows_behind_alone(dev):
    c = _case(10, [40, 7], [5, 2], 16, 2, 128, 16, torch.bfloat16)
    pad = torch.randn(3, 16, 128, dtype=torch.float32).to(torch.bfloat16)
    c["q"] = torch.cat([c["q"], pad])
    c["sets"] += [set()] * 3
    out = torch.full((10, 16, 128), 7.0, dtype=torch.bfloat16, device=dev)
    assert _run(c, dev, out=out) is out
    assert (out[7:] == 7).all() and not (out[:7] == 7).any()


def test_attention_equals_paged_attention_on_chains(dev):
    """A chain is an ordinary chunk: the causal kernels give the same values."""
    from pageserve_b200.paged_attention import paged_attention
    c = _case(11, [500, 33, 1024], [9, 1, 4], 16, 2, 128, 16, torch.bfloat16, kind="chain")
    got = _run(c, dev).double().cpu().numpy()
    ref = paged_attention(c["q"].to(dev), c["k"].to(dev), c["v"].to(dev), _i32(c["tab"], dev), _i32(c["cu"], dev),
                          _i32(c["sp"], dev), c["max_q"], c["max_ctx"]).double().cpu().numpy()
    _, mag = tree.tree_attention(c["q"].double().numpy(), c["k"].double().numpy(), c["v"].double().numpy(), c["tab"],
                                 c["cu"], c["sp"], c["sets"])
    assert (np.abs(got - ref) <= 2 * _tolerance(c, ref, mag)).all()


def test_attention_same_bits_every_time(dev):
    c = _case(12, [3000, 1500], [8, 30], 16, 2, 128, 16, torch.bfloat16)
    a = _run(c, dev)
    for _ in range(3):
        assert torch.equal(a, _run(c, dev))


def test_attention_recorded_errors(dev):
    """Bad metadata skips the request and is recorded; the others are right."""
    c = _case(13, [40, 40, 40], [5, 5, 5], 8, 2, 128, 16, torch.bfloat16)
    good = _run(c, dev)
    t = c["tab"].copy()
    c["tab"][1, 1] = 10 ** 6
    bad = _run(c, dev)
    assert _status() == 1
    assert torch.equal(bad[:5], good[:5]) and torch.equal(bad[10:], good[10:])
    c["tab"] = t
    c["sp"][1] = 10 ** 6
    bad = _run(c, dev, out=torch.zeros_like(good))
    assert _status() == 5
    assert torch.equal(bad[:5], good[:5]) and torch.equal(bad[10:], good[10:]) and (bad[5:10] == 0).all()
    c["sp"][1] = -1
    _run(c, dev)
    assert _status() == 5


def test_attention_streams_and_graph(dev):
    """Another stream than the tensors' own, two workspaces at once, and a
    captured call replayed with new lengths in its buffers."""
    from pageserve_b200 import speculative as sp
    from pageserve_b200.paged_attention import AttentionWorkspace
    c = _case(14, [900, 33], [8, 5], 16, 2, 128, 16, torch.bfloat16)
    want = _run(c, dev)
    q, k, v = (c[x].to(dev) for x in "qkv")
    tab, cu, sp0 = _i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev)
    mask = torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            ws = AttentionWorkspace()
            outs.append([sp.tree_attention(q, k, v, tab, cu, sp0, mask, 8, 928, workspace=ws) for _ in range(20)])
    torch.cuda.synchronize()
    for o in outs[0] + outs[1]:
        assert torch.equal(o, want)
    out = torch.zeros_like(q)
    ws = AttentionWorkspace()
    sp.tree_attention(q, k, v, tab, cu, sp0, mask, 8, 928, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sp.tree_attention(q, k, v, tab, cu, sp0, mask, 8, 928, out=out, workspace=ws)
    g.replay()
    assert torch.equal(out, want)
    sp0.copy_(_i32([411, 12], dev))
    g.replay()
    c["sp"] = [411, 12]
    assert torch.equal(out, _run(c, dev))
    assert _status() == 0


def test_attention_python_refusals(dev):
    from pageserve_b200 import speculative as sp
    c = _case(15, [10], [3], 4, 2, 64, 16, torch.bfloat16)
    q, k, v = (c[x].to(dev) for x in "qkv")
    tab, cu, sp0 = _i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev)
    mask = torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev)
    ok = (q, k, v, tab, cu, sp0, mask, 3, 13)

    def bad(exc, i, x):
        a = list(ok)
        a[i] = x
        with pytest.raises(exc):
            sp.tree_attention(*a)
    bad(TypeError, 0, q.half())
    bad(TypeError, 3, tab.long())
    bad(TypeError, 6, mask.int())
    bad(ValueError, 6, mask.repeat(1, 2))
    bad(ValueError, 6, mask[:2])
    bad(ValueError, 1, k.transpose(0, 1))
    bad(ValueError, 4, cu[:1].clone())
    bad(IndexError, 8, 1000)
    bad(ValueError, 8, 2)
    with pytest.raises(ValueError):
        sp.tree_attention(*ok, out=torch.empty_like(q).transpose(0, 1))
    strided = torch.stack([q, q], -1)[..., 0]  # q in any strides is made contiguous
    assert torch.equal(sp.tree_attention(strided, *ok[1:]), sp.tree_attention(*ok))


def test_attention_cache_past_32_bits(dev):
    """Rows past 2^31 elements of the pool."""
    bs, Hkv, D = 16, 8, 128
    nb = (2 ** 31) // (bs * Hkv * D) + 40
    c = _case(16, [50], [5], 16, Hkv, D, bs, torch.bfloat16)
    n = c["k"].shape[0]
    k = torch.zeros(nb, bs, Hkv, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    k[nb - n:] = c["k"].to(dev)
    v[nb - n:] = c["v"].to(dev)
    small = _run(c, dev)
    c["tab"] = np.where(c["tab"] >= 0, c["tab"] + nb - n, -1)
    c["k"], c["v"] = k, v
    assert torch.equal(_run(c, dev), small)
    assert _status() == 0


def _gpu_reference(c, dev):
    """The oracle's definition (out, sum of weight times |v|) in 64 bits with
    matrix products on the GPU, for sizes where numpy takes minutes."""
    q, k, v = (c[x].to(dev) for x in "qkv")
    hq, d = q.shape[1:]
    hkv, bs = k.shape[2], c["bs"]
    outs, mags = [], []
    for b, n0 in enumerate(c["sp"]):
        a, e = int(c["cu"][b]), int(c["cu"][b + 1])
        n = e - a
        pos = torch.arange(n0 + n, device=dev)
        row = torch.as_tensor(c["tab"][b], device=dev)
        kb, vb = (x[row[pos // bs], pos % bs].double().permute(1, 0, 2) for x in (k, v))  # hkv, keys, d
        qb = q[a:e].double().reshape(n, hkv, hq // hkv, d).permute(1, 2, 0, 3)  # hkv, g, n, d
        s = torch.einsum("hgnd,hkd->hgnk", qb, kb) / np.sqrt(d)
        sees = torch.zeros(n, n, dtype=torch.bool)
        for i, x in enumerate(c["sets"][a:e]):
            sees[i, list(x)] = True
        s[..., n0:].masked_fill_(~sees.to(dev), -float("inf"))
        w = torch.softmax(s, -1)
        outs.append(torch.einsum("hgnk,hkd->hgnd", w, vb).permute(2, 0, 1, 3).reshape(n, hq, d))
        mags.append(torch.einsum("hgnk,hkd->hgnd", w, vb.abs()).permute(2, 0, 1, 3).reshape(n, hq, d))
    return torch.cat(outs), torch.cat(mags)


def _check_large(c, dev, out=None):
    got = (_run(c, dev) if out is None else out).double()
    ref, mag = _gpu_reference(c, dev)
    err, tol = (got - ref).abs(), _tolerance(c, ref.cpu().numpy(), mag.cpu().numpy())
    over = err.cpu().numpy() - tol
    worst = np.unravel_index(np.argmax(over), over.shape)
    assert (over <= 0).all(), (worst, err[worst].item(), tol[worst], ref[worst].item())
    assert _status() == 0


@pytest.mark.parametrize("B,lo,hi,n,heads,dtype", [
    (96, 1000, 1100, 16, (40, 8, 128), torch.bfloat16), (200, 300, 700, 5, (14, 2, 64), torch.float16),
    (64, 130, 260, 8, (16, 2, 128), torch.bfloat16), (6, 700, 2100, 70, (16, 2, 128), torch.float16),
    (40, 1, 500, 33, (8, 8, 128), torch.bfloat16)])
def test_attention_rounds_of_the_ring(dev, B, lo, hi, n, heads, dtype):
    """Enough tiles per CTA that every buffer is used many times, its last tile
    cut anywhere; each row is right and the bits are the same every time."""
    rng = np.random.default_rng(B)
    ctxs = rng.integers(lo, hi + 1, B).tolist()
    c = _case(20, ctxs, [n] * B if n < 30 else rng.integers(1, n + 1, B).tolist(), *heads, 16, dtype)
    a = _run(c, dev)
    for _ in range(6):
        assert torch.equal(a, _run(c, dev))
    _check_large(c, dev, a)


@pytest.mark.parametrize("nodes", [[40, 64, 17, 33], [64] * 3, [128, 1, 100], [256, 16]])
def test_attention_several_row_tiles(dev, nodes):
    _check_large(_case(21, [300, 0, 1023, 64][:len(nodes)], nodes, 16, 2, 128, 16, torch.bfloat16), dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", ["rise", "fall", "spikes"])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(16, 2, 128, 16), (14, 2, 64, 16), (16, 2, 128, 8)])
def test_attention_scores_of_any_size(dev, shape, dtype, Hq, Hkv, D, bs):
    """Scores whose largest rises (or falls, or jumps) by tens from tile to
    tile, so that running sums are rescaled, weights vanish and shares with
    very different maxima are joined."""
    ctxs, nodes = [1500, 700, 130], [9, 20, 3]
    c = _case(22, ctxs, nodes, Hq, Hkv, D, bs, dtype)
    for b, n0 in enumerate(ctxs):
        p = np.arange(n0 + nodes[b])
        grow = {"rise": p / p.size * 20, "fall": (1 - p / p.size) * 20,
                "spikes": np.where(p % 211 == 7, 30.0, 0.05)}[shape]
        blk = torch.as_tensor(c["tab"][b][p // bs])
        rows = c["k"][blk, torch.as_tensor(p % bs)].float() * torch.as_tensor(grow, dtype=torch.float32)[:, None, None]
        c["k"][blk, torch.as_tensor(p % bs)] = rows.to(dtype)
    _check_large(c, dev)


def test_attention_row_that_is_not_finite(dev):
    """A query row of infinities gives NaN, as the formula does, and no other
    row notices."""
    c = _case(23, [700, 60], [5, 3], 16, 2, 128, 16, torch.bfloat16)
    clean = _run(c, dev)
    c["q"][2] = float("inf")
    got = _run(c, dev)
    assert torch.isnan(got[2]).all()
    keep = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("Hq,Hkv,D", [(160, 1, 64), (129, 1, 128)])
def test_attention_wide_groups(dev, Hq, Hkv, D):
    _check_large(_case(24, [50, 300], [3, 9], Hq, Hkv, D, 16, torch.bfloat16), dev)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_alignment_of_out(dev, D):
    c = _case(25, [200, 40], [3, 9], 16, 2, D, 16, torch.bfloat16)
    want = _run(c, dev)
    buf = torch.full((want.numel() + 24,), 5.0, dtype=torch.bfloat16, device=dev)
    out = buf[8:8 + want.numel()].view(want.shape)  # 16- but not 32-byte aligned
    assert torch.equal(_run(c, dev, out=out), want)
    assert (buf[:8] == 5).all() and (buf[8 + want.numel():] == 5).all()
    with pytest.raises(ValueError):
        _run(c, dev, out=buf[1:1 + want.numel()].view(want.shape))


def test_attention_many_calls_in_a_row(dev):
    """Many segments per CTA, thousands of calls queued behind each other: no
    wait runs out (an error is recorded for one that does) and the bits stay."""
    from pageserve_b200 import speculative as sp
    from pageserve_b200.paged_attention import AttentionWorkspace
    rng = np.random.default_rng(28)
    c = _case(28, rng.integers(0, 700, 60).tolist(), rng.integers(1, 20, 60).tolist(), 40, 8, 128, 16, torch.bfloat16)
    want = _run(c, dev)
    q, k, v = (c[x].to(dev) for x in "qkv")
    a = (_i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev),
         torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev), c["max_q"], c["max_ctx"])
    out, ws = torch.zeros_like(q), AttentionWorkspace()
    for _ in range(3000):
        sp.tree_attention(q, k, v, *a, out=out, workspace=ws)
    assert torch.equal(out, want)
    assert _status() == 0


@pytest.mark.parametrize("bs", [48, 80, 96, 192, 384])
@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 64), (16, 2, 128)])
def test_attention_blocks_of_several_boxes(dev, bs, Hq, Hkv, D):
    """Block sizes that are whole 16-key groups but no power of two: keys are
    loaded in the largest power of two that divides them."""
    _check_large(_case(29, [bs - 1, 500, 3 * bs, 1], [7, 20, 1, 3], Hq, Hkv, D, bs, torch.bfloat16), dev)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (14, 2, 64), (40, 8, 128), (64, 1, 64), (3, 1, 128), (33, 1, 64)])
@pytest.mark.parametrize("rows", [64, 65])
def test_attention_small_row_groups(dev, rows, Hq, Hkv, D):
    """On both sides of the bound where rows are doubled, with requests of fewer
    rows, of none and contexts that end anywhere in a tile or are cut."""
    G = Hq // Hkv
    n = max(1, rows // G) + (rows == 65)
    ctxs = [2000, 0, 127, 128, 31, 32, 64, 5000, 96]
    nodes = [n, n, max(1, n - 1), 1, n, 0, n, n, max(1, n // 2)]
    _check_large(_case(30, ctxs, nodes, Hq, Hkv, D, 16, torch.bfloat16, kind="star"), dev)


def test_attention_without_work(dev):
    """Requests that all wait: nothing is written."""
    from pageserve_b200 import speculative as sp
    q = torch.ones(3, 16, 128, dtype=torch.bfloat16, device=dev)
    kv = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16, device=dev)
    out = torch.full_like(q, 3.0)
    mask = torch.zeros(3, 1, dtype=torch.int64, device=dev)
    sp.tree_attention(q, kv, kv, _i32([[0, 1], [2, 3]], dev), _i32([0, 0, 0], dev), _i32([9, 0], dev), mask, 3, 32, out=out)
    assert (out == 3).all() and _status() == 0


def test_attention_refuses_an_output_that_overlaps_q(dev):
    """Every head's rows of q are read by blocks that finish at any time."""
    from pageserve_b200 import speculative as sp
    c = _case(27, [40], [4], 4, 2, 64, 16, torch.bfloat16)
    buf = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=dev)
    buf[:4] = c["q"].to(dev)
    k, v = c["k"].to(dev), c["v"].to(dev)
    mask = torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev)
    a = (k, v, _i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev), mask, 4, 44)
    for lo in (0, 1, 3):
        with pytest.raises(ValueError):
            sp.tree_attention(buf[:4], *a, out=buf[lo:lo + 4])
    assert torch.equal(sp.tree_attention(buf[:4], *a, out=buf[4:]), _run(c, dev))


def test_two_graphs_own_their_scratch(dev):
    """Calls captured without a workspace: two graphs, replayed at once on two
    streams, with shared inputs."""
    from pageserve_b200 import speculative as sp
    c = _case(26, [3000, 1100, 64], [8, 30, 2], 16, 2, 128, 16, torch.bfloat16)
    want = _run(c, dev)
    q, k, v = (c[x].to(dev) for x in "qkv")
    tab, cu, sp0 = _i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev)
    mask = torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sp.tree_attention(q, k, v, tab, cu, sp0, mask, c["max_q"], c["max_ctx"]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    assert _status() == 0


def test_tables_and_acceptance_in_a_graph(dev):
    """A captured step's bookkeeping follows the lengths in its buffers."""
    from pageserve_b200 import speculative as sp
    seq, ql, held = _i32([5, 20], dev), _i32([3, 2], dev), _i32([1, 2], dev)
    tab = _i32([[4, -1, -1], [2, 9, -1]], dev)
    free = _i32([7, 1, 3], dev)
    par = _i32([-1, 0, 0, -1, 0], dev)
    tok = torch.tensor([5, 6, 7, 5, 6], device=dev)
    tgt = _i32([7, 1, 2, 3, 4], dev)

    def step():
        t = sp.build_step_tables(seq, ql, tab, held, free, 10, 16, 5, parents=par, max_q_len=3)
        return t, sp.accept_trees(tok, tgt, t.tree_mask, t.cu_q, seq, 3)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, a = step()
    for s in ([5, 20], [15, 31], [16, 32], [0, 0]):
        seq.copy_(_i32(s, dev))
        held.copy_(_i32([(x + 15) // 16 for x in s], dev))
        g.replay()
        t2, a2 = step()
        for x, y in zip(t + a, t2 + a2):
            assert torch.equal(x, y)
        assert a.num.tolist() == [2, 1] and a.tokens.tolist() == [[7, 2, -1], [3, -1, -1]]
        assert a.start_pos.tolist() == [s[0] + 2, s[1] + 1]
    assert _status() == 0


# -------------------------------------------------------------- accept_trees --

def _check_accept(dev, seed, starts, nodes, agree, L=3, Hkv=2, D=64, bs=16, dtype=torch.bfloat16, vocab=4, kind="random",
                  move=True):
    """Random trees and tokens over a small vocabulary, so that paths of every
    length and ties between siblings with one token occur."""
    from pageserve_b200 import speculative as sp
    rng = np.random.default_rng(seed)
    B = len(starts)
    need = [(s + n + bs - 1) // bs for s, n in zip(starts, nodes)]
    nb = sum(need) + 2
    perm = rng.permutation(nb)
    tab = np.full((B, max(1, max(need))), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        tab[b, :n] = perm[at:at + n]
        at += n
    T = sum(nodes)
    tok, tgt = rng.integers(0, vocab, T), rng.integers(0, vocab, T)
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(int)
    sets, paths = [], []
    for b, n in enumerate(nodes):
        par = _parents(rng, n, kind) if n else []
        for i in range(1, n):
            if rng.random() < agree:
                tok[cu[b] + i] = tgt[cu[b] + par[i]]
        up = tree.ancestors(par)
        sets += up
        paths.append(tree.accept(tok[cu[b]:cu[b + 1]].tolist(), tgt[cu[b]:cu[b + 1]].tolist(), up) if n else [])
    mq = max(1, max(nodes))
    k = torch.randn(L, nb, bs, Hkv, D).to(dtype)
    v = torch.randn(L, nb, bs, Hkv, D).to(dtype)
    kd, vd = k.to(dev), v.to(dev)
    mask = torch.from_numpy(tree.mask_words(sets, (mq + 63) // 64)).to(dev)
    r = sp.accept_trees(torch.from_numpy(tok).to(dev), _i32(tgt, dev), mask, _i32(cu, dev), _i32(starts, dev), mq,
                        *((kd, vd, _i32(tab, dev)) if move else ()))
    assert _status() == 0
    assert r.num.cpu().tolist() == [len(p) for p in paths]
    assert r.start_pos.cpu().tolist() == [s + len(p) for s, p in zip(starts, paths)]
    assert r.nodes.cpu().tolist() == [p + [-1] * (mq - len(p)) for p in paths]
    assert r.tokens.cpu().tolist() == [[int(tgt[cu[b] + j]) for j in p] + [-1] * (mq - len(p))
                                       for b, p in enumerate(paths)]
    for host, devc in ((k, kd), (v, vd)):
        want = host.view(torch.int16 if host.element_size() == 2 else torch.int32).numpy().copy()
        if move:
            for b, p in enumerate(paths):
                tree.move_rows(want, tab[b], bs, starts[b], p)
        assert np.array_equal(devc.cpu().view(torch.int16 if host.element_size() == 2 else torch.int32).numpy(), want)
    return paths


@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 64, 65, 128, 200, 256])
@pytest.mark.parametrize("agree", [0.0, 0.6, 1.0])
def test_accept(dev, n, agree):
    _check_accept(dev, n, [0, 100, 31], [n, max(1, n // 2), n], agree)


@pytest.mark.parametrize("kind", ["chain", "star"])
def test_accept_shapes_of_trees(dev, kind):
    paths = _check_accept(dev, 3, [7, 500], [40, 17], 1.0, kind=kind, vocab=1000)
    assert [len(p) for p in paths] == ([40, 17] if kind == "chain" else [2, 2])


@pytest.mark.parametrize("dtype,Hkv,D,bs,L", [(torch.float16, 1, 64, 4, 1), (torch.float32, 3, 4, 1, 2),
                                              (torch.bfloat16, 8, 128, 64, 5), (torch.bfloat16, 1, 8, 3, 7)])
def test_accept_caches(dev, dtype, Hkv, D, bs, L):
    _check_accept(dev, 4, [0, 13, 64, 3], [9, 0, 20, 1], 0.8, L=L, Hkv=Hkv, D=D, bs=bs, dtype=dtype)


def test_accept_many_requests_and_no_move(dev):
    rng = np.random.default_rng(6)
    _check_accept(dev, 5, rng.integers(0, 50, 200).tolist(), rng.integers(0, 9, 200).tolist(), 0.7, L=1)
    _check_accept(dev, 6, [5, 6], [12, 12], 0.7, move=False)


def test_accept_long_moves_overlap(dev):
    """A deep path one node behind its place: every row moves into its
    neighbour's old place."""
    from pageserve_b200 import speculative as sp
    n = 256
    par = [-1, 0] + [0] + list(range(2, n - 1))  # node 1 is a leaf, 2 .. n-1 a chain below the root
    sets = tree.ancestors(par)
    tgt = np.arange(n)
    tok = np.array([0] + [10 ** 6] + [0] + list(range(2, n - 1)))
    k = torch.arange(2 * 20 * 16 * 8, dtype=torch.float32, device=dev).view(2, 20, 16, 1, 8)
    v = -k
    tab = np.random.default_rng(0).permutation(20)[None]
    want = k.cpu().numpy().copy()
    path = tree.accept(tok.tolist(), tgt.tolist(), sets)
    assert path == [0] + list(range(2, n))
    tree.move_rows(want, tab[0], 16, 21, path)
    r = sp.accept_trees(torch.from_numpy(tok).to(dev), _i32(tgt, dev), torch.from_numpy(tree.mask_words(sets, 4)).to(dev),
                        _i32([0, n], dev), _i32([21], dev), n, k, v, _i32(tab, dev))
    assert int(r.num) == n - 1
    assert np.array_equal(k.cpu().numpy(), want) and np.array_equal(v.cpu().numpy(), -want)


def test_accept_recorded_errors(dev):
    from pageserve_b200 import speculative as sp
    k = torch.zeros(1, 4, 4, 1, 8, device=dev)
    mask = torch.tensor([[1], [3], [5]], device=dev)
    tok, tgt = torch.tensor([0, 9, 5], device=dev), _i32([5, 1, 2], dev)

    def run(cu, start, tab, mq=3):
        m = mask if mq <= 64 else mask.repeat(1, 2)
        r = sp.accept_trees(tok, tgt, m, _i32(cu, dev), _i32(start, dev), mq, k, k.clone(), _i32(tab, dev))
        return r, _status()
    r, e = run([0, 3], [0], [[9, 1]])
    assert e == 1 and r.nodes.cpu().tolist() == [[0, 2, -1]]
    r, e = run([0, 3], [7], [[0, 1]])
    assert e == 5 and int(r.num) == 2
    r, e = run([0, 3], [0], [[0, 1]], mq=2)
    assert e == 5 and int(r.num) == 0 and r.nodes.cpu().tolist() == [[-1, -1]] and int(r.start_pos) == 0
    r, e = run([0, 4], [0], [[0, 1]], mq=4)
    assert e == 5 and int(r.num) == 0


def test_accept_python_refusals(dev):
    from pageserve_b200 import speculative as sp
    k = torch.zeros(1, 4, 4, 1, 8, device=dev)
    mask = torch.tensor([[1], [3], [5]], device=dev)
    tok, tgt, cu, st, tab = (torch.tensor([0, 9, 5], device=dev), _i32([5, 1, 2], dev), _i32([0, 3], dev),
                             _i32([0], dev), _i32([[0, 1]], dev))
    sp.accept_trees(tok, tgt, mask, cu, st, 3, k, k.clone(), tab)
    for exc, a in [(TypeError, (tok.int(), tgt, mask, cu, st, 3)), (TypeError, (tok, tgt.long(), mask, cu, st, 3)),
                   (ValueError, (tok, tgt[:2], mask, cu, st, 3)), (ValueError, (tok, tgt, mask, cu, st, 65)),
                   (ValueError, (tok, tgt, mask, cu, st, 3, k)), (ValueError, (tok, tgt, mask, cu, st, 3, k, k)),
                   (ValueError, (tok, tgt, mask, cu, st, 3, k, k[:, :2].clone(), tab)),
                   (ValueError, (tok, tgt, mask, cu, st, 3, k, k.transpose(2, 3), tab))]:
        with pytest.raises(exc):
            sp.accept_trees(*a)
