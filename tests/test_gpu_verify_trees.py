"""PagedCausalLM.verify_trees: the drafted-tree operators run together around a
model pass, against the one-token-per-step decode of the reference
(engine/runner.py:65-79).

The two paths use different attention kernels and batch shapes, so logits may
differ by the compute dtype's rounding through the model; the bounds are those
of tests/test_gpu_model.py (2e-2 of the largest value for the cache, a greedy
token may differ where the reference margin is below bf16 resolution)."""

import numpy as np
import pytest
import torch

from pageserve_b200 import synthetic

pytestmark = pytest.mark.gpu

REL_TOL = 2e-2


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda", 0)


def near_tie(logits, i):
    top = float(logits.max())
    return top - float(logits[i]) <= 2 ** -7 * abs(top)


def _model(dtype, quant, nb, bs):
    from pageserve_b200.model import PagedCausalLM
    sd = synthetic.generate_state_dict(synthetic.TINY, seed=5, perturb_norms_biases=True)
    m = PagedCausalLM.from_state_dict(sd, synthetic.TINY, device="cuda", dtype=dtype, quantize=quant)
    m.allocate_kv_cache(nb, bs)
    return m


def _draft(rng, root, likely, n, vocab):
    """A tree of n nodes whose first path repeats `likely` for a while, in any
    order that has parents first. -> (tokens, parents)"""
    tokens, parents = [root], [-1]
    tip = 0
    for i in range(1, n):
        if len(likely) and rng.random() < 0.6:  # the next likely token on the path so far
            tokens.append(int(likely[0]))
            parents.append(tip)
            tip, likely = i, likely[1:]
        else:
            tokens.append(int(rng.integers(0, vocab)))
            parents.append(int(rng.integers(0, i)))
    return tokens, parents


class _Requests:
    """The state a serving loop keeps on the device between verified steps."""

    def __init__(self, m, prompts, width, blocks, dev):
        self.m, self.dev, bs = m, dev, m.block_size
        self.seqs = [list(map(int, p)) for p in prompts]  # confirmed tokens; the last is not cached
        self.held = torch.tensor([(len(p) - 1 + bs - 1) // bs for p in prompts], dtype=torch.int32, device=dev)
        tab = np.full((len(prompts), width), -1, np.int32)
        free = list(blocks)
        for b, h in enumerate(self.held.tolist()):
            tab[b, :h] = [free.pop(0) for _ in range(h)]
        self.tables = torch.from_numpy(tab).to(dev)
        self.free = torch.tensor(free, dtype=torch.int32, device=dev)
        self.cached = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=dev)
        lens = self.cached.tolist()
        m.forward_batch(np.concatenate([p[:-1] for p in prompts]), lens, [0] * len(prompts),
                        [row[row >= 0].tolist() for row in tab])

    def take(self, r):
        """Move on by a verified step; -> what it confirmed."""
        num = r.accepted.num.tolist()
        toks = [row[:n] for row, n in zip(r.accepted.tokens.tolist(), num)]
        for s, t in zip(self.seqs, toks):
            s += t
        self.tables, self.held = r.tables.block_tables.clone(), r.tables.held.clone()
        self.free = self.free[int(r.tables.free_used):].clone()
        self.cached = r.accepted.start_pos.clone()
        return toks


@pytest.mark.parametrize("dtype,quant,bs", [(torch.bfloat16, True, 16), (torch.float16, False, 16),
                                            (torch.bfloat16, False, 4)])
def test_verified_trees_decode_as_single_tokens_do(dev, dtype, quant, bs):
    from pageserve_b200 import _lib
    vocab = synthetic.TINY.vocab
    rng = np.random.default_rng(31)
    prompts = [rng.integers(0, vocab, n) for n in (30, 3, 65, 17, 2)]
    B, steps, nb = len(prompts), 9, 400 // bs * 4
    m = _model(dtype, quant, nb, bs)
    _lib.device_status(clear=True)
    # one token per step: what the drafts are made of
    width = 256 // bs
    tabs = [list(range(b * width, (b + 1) * width)) for b in range(B)]
    m.forward_batch(np.concatenate([p[:-1] for p in prompts]), [len(p) - 1 for p in prompts], [0] * B, tabs)
    likely = [[int(p[-1])] for p in prompts]
    for i in range(60):
        _, nxt = m.forward_batch([t[-1] for t in likely], [1] * B, [len(p) - 1 + i for p in prompts], tabs)
        for t, x in zip(likely, nxt.tolist()):
            t.append(x)
    m.allocate_kv_cache(nb, bs)
    s = _Requests(m, prompts, width + 3, rng.permutation(nb).tolist(), dev)
    confirmed = 0
    for step in range(steps):
        rows, pars, qs = [], [], []
        for b in range(B):
            done = len(s.seqs[b]) - len(prompts[b])
            n = 0 if (step + b) % 7 == 6 else int(rng.integers(1, 12))  # now and then a request waits
            t, p = _draft(rng, s.seqs[b][-1], likely[b][done + 1:], n, vocab) if n else ([], [])
            rows, pars, qs = rows + t, pars + p, qs + [n]
        pad = int(rng.integers(0, 4))
        r = m.verify_trees(torch.tensor(rows + [0] * pad, device=dev),
                           torch.tensor(pars + [-1] * pad, dtype=torch.int32, device=dev), s.cached,
                           torch.tensor(qs, dtype=torch.int32, device=dev), s.tables, s.held, s.free, 11,
                           return_logits=step % 2 == 0)
        assert (r.logits is not None) == (step % 2 == 0)
        toks = s.take(r)
        assert [len(t) > 0 for t in toks] == [n > 0 for n in qs]
        confirmed += sum(map(len, toks))
    assert _lib.device_status(clear=True) == 0
    assert confirmed > 1.5 * steps * B  # drafts were taken
    assert s.cached.tolist() == [len(x) - 1 for x in s.seqs]
    # every confirmed token is the greedy one, and the cache holds its sequence
    from pageserve_b200.paged_attention import gather_kv
    own = m.k_cache, m.v_cache
    m.allocate_kv_cache(nb, bs)
    for b in range(B):
        seq, n0 = s.seqs[b], len(prompts[b])
        n = len(seq) - 1
        lg = m.forward_step(torch.tensor(seq[:-1]), list(range(width)), 0).float()
        for i in range(n0 - 1, n):
            assert int(lg[i].argmax()) == seq[i + 1] or near_tie(lg[i], seq[i + 1]), (b, i)
        for layer in range(m.k_cache.shape[0]):
            want = gather_kv(m.k_cache[layer], m.v_cache[layer], list(range(width)), bs, n)
            got = gather_kv(own[0][layer], own[1][layer], s.tables[b], bs, n)
            for x, y in zip(got, want):
                assert float((x.float() - y.float()).abs().max()) <= REL_TOL * float(y.float().abs().max()), (b, layer)


def test_captured_verification(dev):
    """A step captured once and replayed with new trees and lengths yields what
    the call itself does, bit for bit."""
    vocab, bs, nb = synthetic.TINY.vocab, 16, 64
    rng = np.random.default_rng(32)
    prompts = [rng.integers(0, vocab, n) for n in (40, 9, 22)]
    qs = torch.tensor([6, 5, 7], dtype=torch.int32, device=dev)
    drafts = [[_draft(np.random.default_rng([i, b]), 0, [], n, vocab) for b, n in enumerate(qs.tolist())]
              for i in range(5)]
    results = []
    for mode in ("call", "graph"):
        m = _model(torch.bfloat16, True, nb, bs)
        s = _Requests(m, prompts, 12, range(nb), dev)
        tok = torch.zeros(18, dtype=torch.int64, device=dev)
        par = torch.zeros(18, dtype=torch.int32, device=dev)
        cached, tables, held = s.cached.clone(), s.tables.clone(), s.held.clone()
        free = torch.arange(nb - 12, nb, dtype=torch.int32, device=dev)
        graph, out = None, []
        for step in drafts:
            t = sum(([s.seqs[b][-1]] + d[0][1:] for b, d in enumerate(step)), [])
            tok.copy_(torch.tensor(t))
            par.copy_(torch.tensor(sum((d[1] for d in step), []), dtype=torch.int32))
            if mode == "graph" and graph is None:
                keep = m.k_cache.clone(), m.v_cache.clone()
                m.verify_trees(tok, par, cached, qs, tables, held, free, 7, 192)  # loads kernels, sizes workspaces
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    r = m.verify_trees(tok, par, cached, qs, tables, held, free, 7, 192, return_logits=True)
                m.k_cache.copy_(keep[0])
                m.v_cache.copy_(keep[1])
            if mode == "graph":
                graph.replay()
            else:
                r = m.verify_trees(tok, par, cached, qs, tables, held, free, 7, 192, return_logits=True)
            toks = [row[:n] for row, n in zip(r.accepted.tokens.tolist(), r.accepted.num.tolist())]
            for x, y in zip(s.seqs, toks):
                x += y
            out += [r.logits.clone(), r.targets.clone(), r.accepted.nodes.clone()]
            cached.copy_(r.accepted.start_pos)
            tables.copy_(r.tables.block_tables)
            held.copy_(r.tables.held)
            free.copy_(torch.cat([free[int(r.tables.free_used):], free[:int(r.tables.free_used)]]))
        results.append((out, m.k_cache, m.v_cache, s.seqs))
        if graph is not None:
            graph.reset()
    assert results[0][3] == results[1][3]
    for x, y in zip(results[0][0], results[1][0]):
        assert torch.equal(x, y)
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])


def test_verification_refusals(dev):
    m = _model(torch.bfloat16, True, 16, 16)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    one = torch.ones_like(i)
    par = torch.full_like(i, -1)
    tab = torch.full((1, 2), -1, dtype=torch.int32, device=dev)
    tok = torch.zeros(1, dtype=torch.int64, device=dev)
    free = torch.arange(4, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        m.verify_trees(tok.int(), par, i, one, tab, i, free, 1)
    with pytest.raises(TypeError):
        m.verify_trees(torch.zeros(4, dtype=torch.int64, device=dev)[::2], par, i, one, tab, i, free, 1)
    with pytest.raises(RuntimeError):
        m.verify_trees(tok.cpu(), par, i, one, tab, i, free, 1)
    with pytest.raises(ValueError):
        m.verify_trees(tok[:0], par, i, one, tab, i, free, 1)
    with pytest.raises(ValueError):
        m.verify_trees(torch.zeros(2, dtype=torch.int64, device=dev), par, i, one, tab, i, free, 1)
    with pytest.raises(ValueError):
        m.verify_trees(tok, par, i, one, tab, i, free, 0)
    with pytest.raises(NotImplementedError):
        m.verify_trees(tok, par, i, one, tab, i, free, 257)
    with pytest.raises(IndexError):
        m.verify_trees(tok, par, i, one, tab, i, free, 1, max_ctx=33)
    r = m.verify_trees(tok, par, i, one, tab, i, free, 1)
    assert r.accepted.num.tolist() == [1] and r.accepted.start_pos.tolist() == [1]
    m.k_cache = None
    with pytest.raises(RuntimeError):
        m.verify_trees(tok, par, i, one, tab, i, free, 1)


def test_all_requests_wait(dev):
    """A step of padding alone changes nothing."""
    from pageserve_b200 import _lib
    m = _model(torch.bfloat16, True, 16, 16)
    s = _Requests(m, [np.arange(20), np.arange(5)], 4, range(16), dev)
    before = m.k_cache.clone(), m.v_cache.clone()
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    r = m.verify_trees(torch.zeros(3, dtype=torch.int64, device=dev), torch.full((3,), -1, dtype=torch.int32, device=dev),
                       s.cached, zero, s.tables, s.held, s.free, 8)
    assert s.take(r) == [[], []] and s.cached.tolist() == [19, 4]
    assert torch.equal(m.k_cache, before[0]) and torch.equal(m.v_cache, before[1])
    assert _lib.device_status(clear=True) == 0
