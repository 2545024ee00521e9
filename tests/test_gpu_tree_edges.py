"""Drafted-tree operators where a step cannot be carried out in full, where
cached values are not finite, and how far results may be off on average."""

import numpy as np
import pytest
import torch

from oracle import tree
from test_gpu_speculative import _case, _gpu_reference, _i32, _run, _status, dev  # noqa: F401
from test_gpu_verify_trees import _model, _Requests, near_tie

pytestmark = pytest.mark.gpu


# ------------------------------------------- steps that are not stored whole --

def _greedy(m, prompts, n):
    """Each prompt's n greedy tokens, one per step."""
    B, width = len(prompts), 128 // m.block_size
    tabs = [list(range(b * width, (b + 1) * width)) for b in range(B)]
    _, nxt = m.forward_batch(np.concatenate(prompts), [len(p) for p in prompts], [0] * B, tabs)
    out = [[int(x)] for x in nxt.tolist()]
    for i in range(n - 1):
        _, nxt = m.forward_batch([t[-1] for t in out], [1] * B, [len(p) + i for p in prompts], tabs)
        for t, x in zip(out, nxt.tolist()):
            t.append(x)
    m.allocate_kv_cache(m.num_blocks, m.block_size)
    return out


def _verify_chains(s, drafts, **kw):
    """One step of chains: every request's last confirmed token and its draft."""
    rows, pars, qs = [], [], []
    for seq, d in zip(s.seqs, drafts):
        rows += [seq[-1]] + d
        pars += range(-1, len(d))
        qs.append(1 + len(d))
    return s.m.verify_trees(torch.tensor(rows, device=s.dev), torch.tensor(pars, dtype=torch.int32, device=s.dev),
                            s.cached, torch.tensor(qs, dtype=torch.int32, device=s.dev), s.tables, s.held, s.free,
                            max(qs), **kw)


def _check_sequences(s, prompts):
    """Every confirmed token is the greedy one of a pass over the sequence."""
    m, bs = s.m, s.m.block_size
    m.allocate_kv_cache(m.num_blocks, bs)
    for seq, p in zip(s.seqs, prompts):
        lg = m.forward_step(torch.tensor(seq[:-1]), list(range(128 // bs)), 0).float()
        for i in range(len(p) - 1, len(seq) - 1):
            assert int(lg[i].argmax()) == seq[i + 1] or near_tie(lg[i], seq[i + 1]), i


@pytest.fixture()
def two_requests(dev):  # noqa: F811
    """Blocks of 4: request 0 has 8 tokens cached in 2 blocks (its next row
    needs a third), request 1 has 5 in 2 (room for 3 rows); and what the model
    goes on with."""
    m = _model(torch.bfloat16, False, 64, 4)
    prompts = [np.arange(3, 12), np.arange(40, 46)]
    likely = _greedy(m, prompts, 12)
    _status()
    return _Requests(m, prompts, 8, range(64), dev), prompts, likely


def test_verification_with_a_short_free_list(two_requests):
    """Rows that get no block are stored nowhere: nothing of them is kept, and
    the next step goes on from what is."""
    s, prompts, likely = two_requests
    free, s.free = s.free, s.free[:0]
    r = _verify_chains(s, [x[:4] for x in likely])
    assert _status() == 6
    assert int(r.tables.free_used) == 3  # 13 positions and 10 in blocks of 4: 4 and 3, 2 held each
    num, start = r.accepted.num.tolist(), r.accepted.start_pos.tolist()
    assert num[0] == 0 and start[0] == 8 and r.accepted.tokens[0].tolist() == [-1] * 5
    assert 1 <= num[1] <= 3 and start[1] == 5 + num[1]
    assert all(p <= h * 4 for p, h in zip(start, r.tables.held.tolist()))
    s.take(r._replace(tables=r.tables._replace(free_used=torch.zeros(1))))
    s.free = free
    for _ in range(2):
        done = [len(q) - len(p) for q, p in zip(s.seqs, prompts)]
        r = _verify_chains(s, [x[n:n + 3] for x, n in zip(likely, done)])
        assert min(r.accepted.num.tolist()) >= 1
        s.take(r)
    assert _status() == 0
    assert s.cached.tolist() == [len(x) - 1 for x in s.seqs]
    _check_sequences(s, prompts)


def test_tables_rows_without_a_slot_see_nothing(dev):  # noqa: F811
    """Behind the first row without a slot nothing can be kept: masks are 0."""
    from pageserve_b200 import speculative as sp

    def run(seq, q, tab, held, free, par, mq, **kw):
        r = sp.build_step_tables(_i32(seq, dev), _i32(q, dev), _i32(tab, dev), _i32(held, dev), _i32(free, dev), 9, 4,
                                 len(par), parents=_i32(par, dev), max_q_len=mq, **kw)
        return r.slots.tolist(), [[int(x) & (2 ** 64 - 1) for x in row] for row in r.tree_mask.tolist()], \
            r.positions.tolist(), _status()
    # one block for the two that the second request needs
    slots, mask, pos, e = run([2, 3], [2, 6], [[4, -1, -1], [7, -1, -1]], [1, 1], [5], [-1, 0, -1, 0, 1, 0, 0, 3], 6)
    assert slots == [18, 19, 31, 20, 21, 22, 23, -1] and e == 6
    assert [m[0] for m in mask] == [1, 3, 1, 3, 7, 9, 17, 0]
    assert pos == [2, 3, 3, 4, 5, 4, 4, 5]
    # a held block outside the pool: rows behind it that have a place count as little
    slots, mask, pos, e = run([3], [6], [[4, 99, 2]], [3], [], [-1, -1, 0, 1, 0, 2], 6)
    assert slots == [19, -1, -1, -1, -1, 8] and e == 1
    assert [m[0] for m in mask] == [1, 0, 0, 0, 0, 0]
    # past the table: attention leaves the whole request out
    slots, mask, pos, e = run([6, 1], [3, 2], [[4, 1], [7, -1]], [2, 1], [], [-1, 0, 1, -1, 0], 3)
    assert slots == [6, 7, -1, 29, 30] and e == 5
    assert [m[0] for m in mask] == [0, 0, 0, 1, 3]
    # several words, the rows without a slot in the middle of a warp
    n = 100
    slots, mask, pos, e = run([0], [n], [[-1] * 25], [0], range(9), list(range(-1, n - 1)), n)
    assert e == 6 and slots == list(range(36)) + [-1] * 64
    assert mask == [[2 ** (i + 1) - 1, 0] for i in range(36)] + [[0, 0]] * 64


def test_acceptance_counts_cached_rows_only(dev):  # noqa: F811
    """start_pos ends where the table has no block for a row of the path or
    for its place, whatever the model agrees with."""
    from pageserve_b200 import speculative as sp
    sets = tree.ancestors([-1, 0, 0, 2, 3, 4])  # the path 0 2 3 4 5
    tgt = [1, 9, 2, 3, 4, 5]
    tok = [0, 8, 1, 2, 3, 4]
    k = torch.arange(2 * 6 * 2 * 8, dtype=torch.float32, device=dev).view(2, 6, 2, 1, 8)

    def run(start, tab):
        kc, vc = k.clone(), -k
        r = sp.accept_trees(torch.tensor(tok, device=dev), _i32(tgt, dev), torch.from_numpy(tree.mask_words(sets, 1)).to(dev),
                            _i32([0, 6], dev), _i32([start], dev), 6, kc, vc, _i32([tab], dev))
        assert r.nodes.tolist() == [[0, 2, 3, 4, 5, -1]] and int(r.num) == 5
        kept = int(r.start_pos) - start
        want = k.cpu().numpy().copy()
        tree.move_rows(want, tab, 2, start, [0, 2, 3, 4, 5][:kept])
        assert np.array_equal(kc.cpu().numpy(), want) and np.array_equal(vc.cpu().numpy(), -want)
        return kept, _status()
    assert run(0, [3, 1, 4]) == (5, 0)
    assert run(2, [5, 3, 1, 4]) == (5, 0)
    assert run(0, [9, 1, 4]) == (0, 1)      # the root's own block
    assert run(0, [3, -1, 4]) == (1, 1)     # node 2's
    assert run(0, [3, 1, 6]) == (3, 1)      # node 4's
    assert run(1, [3, 1, 0]) == (4, 5)      # node 5 is past the table
    assert run(5, [9, 9, 2]) == (1, 5)
    assert run(6, [0, 1, 2]) == (0, 5)


def test_verification_past_the_bounds_keeps_nothing(two_requests):
    """A request whose context passes max_ctx, or its row of the table, is
    left out by the attention: nothing of it is kept, the others are right."""
    s, prompts, likely = two_requests
    r = _verify_chains(s, [x[:4] for x in likely], max_ctx=12)  # contexts 13 and 10
    assert _status() == 5
    assert r.accepted.num[0] == 0 and r.accepted.start_pos[0] == 8
    assert r.accepted.nodes[0].tolist() == [-1] * 5 and r.accepted.tokens[0].tolist() == [-1] * 5
    assert r.accepted.num[1] >= 1
    s.take(r)
    wide, s.tables = s.tables, s.tables[:, :3].contiguous()  # 12 positions
    done = len(s.seqs[1]) - len(prompts[1])
    r = _verify_chains(s, [likely[0][:4], likely[1][done:done + 1]])
    assert _status() == 5
    assert r.accepted.num[0] == 0 and r.accepted.start_pos[0] == 8 and r.accepted.num[1] >= 1
    s.take(r)
    s.tables = torch.cat([s.tables, wide[:, 3:]], 1)
    for _ in range(2):
        done = [len(q) - len(p) for q, p in zip(s.seqs, prompts)]
        s.take(_verify_chains(s, [x[n:n + 2] for x, n in zip(likely, done)], max_ctx=20))
    assert _status() == 0
    _check_sequences(s, prompts)


def test_padding_rows_are_the_same_every_time(dev):  # noqa: F811
    """Rows behind the last request have defined results, whatever the memory
    held before."""
    m = _model(torch.bfloat16, True, 16, 16)
    s = _Requests(m, [np.arange(20), np.arange(5)], 4, range(16), dev)
    tok = torch.arange(9, device=dev)
    par = torch.full((9,), -1, dtype=torch.int32, device=dev)
    q = torch.ones(2, dtype=torch.int32, device=dev)
    got = []
    for fill in (float("nan"), 3.0):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        junk = [torch.full((2 ** k,), fill, dtype=torch.bfloat16, device=dev) for k in range(8, 22) for _ in range(4)]
        del junk
        got.append(m.verify_trees(tok, par, s.cached, q, s.tables, s.held, s.free, 1, return_logits=True))
    for r in got:
        assert torch.isfinite(r.logits).all()
    assert torch.equal(got[0].logits, got[1].logits) and torch.equal(got[0].targets, got[1].targets)
    assert _status() == 0


LO, HI = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("cu", [[HI - 2, LO + 2], [LO, LO + 3], [HI - 2, HI], [-1, 2], [4, 9], [3, 1], [LO, HI], [HI, LO]])
def test_row_offsets_of_any_value(dev, cu):  # noqa: F811
    """Row offsets that are out of range, or whose difference wraps to a small
    number, are recorded and skipped."""
    from pageserve_b200 import speculative as sp
    c = _case(44, [30], [7], 16, 2, 128, 16, torch.bfloat16)
    c["max_q"], c["cu"] = 7, np.asarray(cu)
    for bs in (16, 4):
        c["bs"] = bs
        out = torch.full((7, 16, 128), 7.0, dtype=torch.bfloat16, device=dev)
        _run(c, dev, out=out)
        assert (out == 7).all() and _status() == 5
        c["k"], c["v"] = (x.reshape(-1, 4, 2, 128) for x in (c["k"], c["v"]))
        c["tab"] = np.zeros((1, 12), int)
    k = torch.randn(1, 4, 4, 1, 8, device=dev)
    v, k0 = -k, k.clone()
    mask = torch.tensor([[(2 << i) - 1] for i in range(7)], device=dev)
    tok = torch.zeros(7, dtype=torch.int64, device=dev)
    r = sp.accept_trees(tok, tok.int(), mask, _i32(cu, dev), _i32([3], dev), 7, k, v, _i32([[0, 1, 2]], dev))
    assert _status() == 5
    assert r.num.tolist() == [0] and r.start_pos.tolist() == [3]
    assert r.nodes.tolist() == [[-1] * 7] and r.tokens.tolist() == [[-1] * 7]
    assert torch.equal(k, k0) and torch.equal(v, -k0)


def test_start_positions_of_any_value(dev):  # noqa: F811
    """A start whose sum with the rows passes 32 bits, and one below 0."""
    from pageserve_b200 import speculative as sp
    mask = torch.tensor([[(2 << i) - 1] for i in range(3)], device=dev)
    tok = torch.zeros(3, dtype=torch.int64, device=dev)
    for start in (HI, HI - 2, -1, LO):
        for caches in ((), (torch.zeros(1, 4, 4, 1, 8, device=dev), torch.zeros(1, 4, 4, 1, 8, device=dev),
                            _i32([[0, 1]], dev))):
            r = sp.accept_trees(tok, tok.int(), mask, _i32([0, 3], dev), _i32([start], dev), 3, *caches)
            assert _status() == 5
            assert r.num.tolist() == [0] and r.start_pos.tolist() == [start] and r.tokens.tolist() == [[-1] * 3]
    r = sp.accept_trees(tok, tok.int(), mask, _i32([0, 3], dev), _i32([HI - 3], dev), 3)
    assert _status() == 0 and r.num.tolist() == [3] and r.start_pos.tolist() == [HI]


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


@pytest.mark.parametrize("D,bs,nodes", [(128, 16, 6), (64, 16, 20), (128, 4, 6)])
def test_attention_infinities_in_the_cache_and_in_a_node(dev, D, bs, nodes):  # noqa: F811
    """Rows that see the node get NaN of both signs, the others keep the cache's."""
    for ctx in (50, 900):
        c = _case(47, [ctx, 40], [nodes, 5], 8, 2, D, bs, torch.bfloat16)
        sees = torch.tensor([2 in x for x in c["sets"][:nodes]])
        col = _with_value(c, dev, [(ctx // 3, float("-inf")), (ctx + 2, float("inf"))], 4)
        assert torch.isnan(col[sees]).all() and (col[~sees] == float("-inf")).all()
        assert sees.any() and not sees.all()


@pytest.mark.parametrize("D,bs,n", [(128, 16, 8), (64, 16, 40), (128, 4, 8)])
def test_attention_many_infinities(dev, D, bs, n):  # noqa: F811
    """Every row of many segments of a CTA is looked at again."""
    rng = np.random.default_rng(48)
    c = _case(48, rng.integers(1, 900, 60).tolist(), [n] * 60, 40, 8, D, bs, torch.bfloat16)
    for b in range(60):
        c["v"][c["tab"][b, 0], 0] = float("inf")
    for _ in range(3):
        assert torch.isposinf(_run(c, dev)).all()
    assert _status() == 0


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


# ------------------------------------------------------- errors on average --

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ctxs,nodes,Hq,Hkv,D,bs", [
    ([300, 5, 511], [33, 64, 1], 16, 2, 128, 16), ([700, 130, 64], [7, 8, 2], 16, 2, 128, 16),
    ([5000, 1, 2048, 700], [3, 1, 8, 11], 14, 2, 64, 16), ([900, 77], [12, 50], 40, 8, 128, 4),
    ([6000], [40], 40, 8, 128, 16)])
def test_attention_error_on_average(dev, ctxs, nodes, Hq, Hkv, D, bs, dtype):  # noqa: F811
    """Roundings are independent, so their mean square adds up. With u half a
    step of the type: rounding a weight w is off by at most u w and, spread
    evenly, by u w / sqrt(3) in the mean, and so is the output o. The mean of
    err^2 / (u^2 / 3 (sum w^2 v^2 + o^2)) is then at most 1 and, as a value lies
    anywhere between two powers of two, about 1/2 (half steps are between u/2 and
    u of a value). f16 weights of 2^-14 of the reference power or less are off
    by up to 2^-25 of it, the sum being at least 1/2 of it: 2^-24 v each. Scores
    are off by a few 2^-22, below 1% of u. So the root is below 1; a second
    rounding of P, or f16 weights taken through bf16, would give 1.2 or 8."""
    c = _case(43, ctxs, nodes, Hq, Hkv, D, bs, dtype)
    got = _run(c, dev).double()
    ref, _ = _gpu_reference(c, dev)
    sq, count = _gpu_squares(c, dev)
    u = torch.finfo(dtype).eps / 2
    var = u * u / 3 * (sq + ref * ref)
    if dtype == torch.float16:
        var = var + count * (2.0 ** -24) ** 2 / 3
    z = float(((got - ref) ** 2 / var).mean().sqrt())
    assert z < 1.0, z
    assert _status() == 0


def _gpu_squares(c, dev):  # noqa: F811
    """Of every output: the sum of w^2 v^2, and the sum of v^2 of the weights
    that 16 bits hold with a fixed step, in 64 bits."""
    q, k, v = (c[x].to(dev) for x in "qkv")
    hq, d = q.shape[1:]
    hkv, bs = k.shape[2], c["bs"]
    sqs, counts = [], []
    for b, n0 in enumerate(c["sp"]):
        a, e = int(c["cu"][b]), int(c["cu"][b + 1])
        n = e - a
        pos = torch.arange(n0 + n, device=dev)
        row = torch.as_tensor(c["tab"][b], device=dev)
        kb, vb = (x[row[pos // bs], pos % bs].double().permute(1, 0, 2) for x in (k, v))
        qb = q[a:e].double().reshape(n, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        s = torch.einsum("hgnd,hkd->hgnk", qb, kb) / np.sqrt(d)
        sees = torch.zeros(n, n, dtype=torch.bool)
        for i, x in enumerate(c["sets"][a:e]):
            sees[i, list(x)] = True
        s[..., n0:].masked_fill_(~sees.to(dev), -float("inf"))
        w = torch.softmax(s, -1)
        small = ((w < 2.0 ** -13) & (w > 0)).double()
        sqs.append(torch.einsum("hgnk,hkd->hgnd", w * w, vb * vb).permute(2, 0, 1, 3).reshape(n, hq, d))
        counts.append(torch.einsum("hgnk,hkd->hgnd", small, vb * vb).permute(2, 0, 1, 3).reshape(n, hq, d))
    return torch.cat(sqs), torch.cat(counts)


# ------------------------------------------------------------- the operators --

def test_outputs_are_tensors_of_their_own(dev):  # noqa: F811
    """No two outputs share a storage: what a caller keeps for the next step
    holds no other output, and tracing may free each by itself."""
    from pageserve_b200 import speculative as sp
    i, tab = _i32([3, 5], dev), _i32([[0, -1], [1, -1]], dev)
    t = sp.build_step_tables(i, _i32([2, 1], dev), tab, _i32([1, 1], dev), _i32([2, 3], dev), 4, 16, 3,
                             parents=_i32([-1, 0, -1], dev), max_q_len=2)
    a = sp.accept_trees(torch.tensor([1, 2, 3], device=dev), _i32([2, 3, 4], dev), t.tree_mask, t.cu_q, i, 2)
    for outs in (t, a, sp.build_step_tables(i, _i32([2, 1], dev), tab, _i32([1, 1], dev), _i32([2, 3], dev), 4, 16, 3)):
        outs = [x for x in outs if x is not None]
        assert len({x.untyped_storage().data_ptr() for x in outs}) == len(outs)
        assert all(x.untyped_storage().nbytes() == x.numel() * x.element_size() for x in outs)


def test_captured_call_keeps_its_scratch(dev):  # noqa: F811
    """A graph that was captured with a workspace goes on being right when a
    larger call has outgrown it, and writes nowhere else."""
    from pageserve_b200 import speculative as sp
    from pageserve_b200.paged_attention import AttentionWorkspace
    c = _case(45, [700, 300], [8, 30], 16, 2, 128, 16, torch.bfloat16)
    want = _run(c, dev)
    q, k, v = (c[x].to(dev) for x in "qkv")
    a = (_i32(c["tab"], dev), _i32(c["cu"], dev), _i32(c["sp"], dev),
         torch.from_numpy(tree.mask_words(c["sets"], 1)).to(dev), 30, 708)
    out, ws = torch.zeros_like(q), AttentionWorkspace()
    sp.tree_attention(q, k, v, *a, out=out, workspace=ws)
    size = ws.buf.numel()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sp.tree_attention(q, k, v, *a, out=out, workspace=ws)
    big = _case(46, [5000] * 8, [40] * 8, 40, 8, 128, 16, torch.bfloat16)
    for _ in range(2):
        _run(big, dev, workspace=ws)
    assert ws.buf.numel() > size
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    other = [torch.full((size,), 77, dtype=torch.uint8, device=dev) for _ in range(4)]
    out.zero_()
    g.replay()
    assert torch.equal(out, want)
    assert all((x == 77).all() for x in other)
    assert _status() == 0
