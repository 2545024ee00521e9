"""The operators of decoding with drafted token trees, as cases to measure.

Three operators over the paged KV cache, in the order a step uses them:

* ``tables``  block tables, positions, KV slots and ancestor masks of a step,
  from the requests' lengths, their drafted trees and the list of free blocks;
* ``attn``    attention of the drafted nodes over the cached context and their
  own ancestors;
* ``accept``  the longest drafted path the model agrees with, and the move of
  its keys and values to the places they keep in the cache.

``run`` computes an operator in its plain form (elementary torch operations,
32 bits) or, where ``own`` is true, by the framework's entry points.

Conventions: B requests; request b has ``seq_lens[b]`` tokens in the cache and
``q_lens[b]`` new ones in this step, rows ``cu_q[b] .. cu_q[b+1]``. New token i
of a request is stored at cache position ``seq_lens[b] + i``; as a tree node it
has a parent among the earlier ones (-1: none) and sits, for the rotary
embedding, at position ``seq_lens[b] + depth``. Bit j % 64 of word j // 64 of
its mask row says that node j is an ancestor of it, or itself.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
VOCAB = 151936


def listed():
    return [
        # one request decoding its next token: the latency of a step's bookkeeping
        {"name": "tables_one_request", "op": "tables", "B": 1, "ctx_lo": 37, "ctx_hi": 37, "nodes": 1, "tree": False,
         "bs": 16, "width": 16, "chunk": 0, "fresh": False},
        # an ordinary batch of drafted trees of up to 16 nodes
        {"name": "tables_trees_64", "op": "tables", "B": 64, "ctx_lo": 1900, "ctx_hi": 2048, "nodes": 16, "tree": True,
         "bs": 16, "width": 256, "chunk": 0, "fresh": False},
        # a large mixed step: many decoding requests of any length up to 32k and some prompt chunks,
        # their tables rebuilt from the lengths
        {"name": "tables_mixed_513", "op": "tables", "B": 513, "ctx_lo": 0, "ctx_hi": 32000, "nodes": 1, "tree": False,
         "bs": 16, "width": 2049, "chunk": 509, "fresh": True},
        # one request, a single new token on a short context: the smallest call
        {"name": "attn_one_node", "op": "attn", "B": 1, "Hq": 14, "Hkv": 2, "D": 64, "ctx_lo": 128, "ctx_hi": 128,
         "nodes": 1, "ragged": False, "bs": 16, "dtype": "bf16"},
        # a few requests of a small model with ragged little trees
        {"name": "attn_small_f16", "op": "attn", "B": 5, "Hq": 14, "Hkv": 2, "D": 64, "ctx_lo": 37, "ctx_hi": 511,
         "nodes": 7, "ragged": True, "bs": 16, "dtype": "f16"},
        # the ordinary serving batch: 64 requests at context 2048, 8 nodes each
        {"name": "attn_64x8", "op": "attn", "B": 64, "Hq": 16, "Hkv": 2, "D": 128, "ctx_lo": 2048, "ctx_hi": 2048,
         "nodes": 8, "ragged": False, "bs": 16, "dtype": "bf16"},
        # few requests with wide trees on uneven contexts
        {"name": "attn_8x64_ragged", "op": "attn", "B": 8, "Hq": 16, "Hkv": 2, "D": 128, "ctx_lo": 512, "ctx_hi": 4096,
         "nodes": 64, "ragged": True, "bs": 16, "dtype": "bf16"},
        # one request on a long context: the work has to be split along it
        {"name": "attn_long_f16", "op": "attn", "B": 1, "Hq": 40, "Hkv": 8, "D": 128, "ctx_lo": 32717,
         "ctx_hi": 32717, "nodes": 33, "ragged": False, "bs": 16, "dtype": "f16"},
        # the largest: 128 requests at context 4096 of a large model, 16 nodes each
        {"name": "attn_128x16", "op": "attn", "B": 128, "Hq": 40, "Hkv": 8, "D": 128, "ctx_lo": 4000, "ctx_hi": 4096,
         "nodes": 16, "ragged": False, "bs": 16, "dtype": "bf16"},
        # one request of a small model: the latency of accepting a little tree
        {"name": "accept_one_f16", "op": "accept", "B": 1, "layers": 24, "Hkv": 2, "D": 64, "ctx_lo": 130,
         "ctx_hi": 130, "nodes": 7, "accepted": 3, "bs": 16, "dtype": "f16"},
        # the ordinary serving batch
        {"name": "accept_64x16", "op": "accept", "B": 64, "layers": 36, "Hkv": 2, "D": 128, "ctx_lo": 1900,
         "ctx_hi": 2048, "nodes": 16, "accepted": 4, "bs": 16, "dtype": "bf16"},
        # a deep cache and wide trees, several tokens kept
        {"name": "accept_32x61", "op": "accept", "B": 32, "layers": 64, "Hkv": 8, "D": 128, "ctx_lo": 500,
         "ctx_hi": 4096, "nodes": 61, "accepted": 7, "bs": 16, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tables", "attn", "attn", "accept"])
    if op == "tables":
        tree = rng.random() < 0.5
        hi = _spread(rng, 20, 32000)
        bs = rng.choice([1, 8, 16, 16, 16, 24, 32, 64])
        nodes = _spread(rng, 2, 200) if tree else 1
        chunk = 0 if tree else rng.choice([0, _spread(rng, 8, 509)])
        need = (hi + max(nodes, chunk) + bs - 1) // bs
        B = _spread(rng, 1, 513)
        B = min(B, max(1, 1000000 // need))
        return {"op": op, "B": B, "ctx_lo": rng.randint(0, hi), "ctx_hi": hi, "nodes": nodes, "tree": tree, "bs": bs,
                "width": need + rng.randint(0, 9), "chunk": chunk, "fresh": rng.random() < 0.4}
    Hq, Hkv, D = rng.choice([(14, 2, 64), (16, 2, 128), (40, 8, 128), (4, 4, 64), (8, 8, 128), (16, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "attn":
        B = _spread(rng, 1, 128)
        hi = _spread(rng, 1, 32768)
        nodes = _spread(rng, 1, 130)
        # within the largest listed case's work: 128 requests x 4096 keys x 8 kv heads x 128, 16 nodes x 40 heads
        while B * (hi + nodes) * max(Hkv * D / 1024.0, nodes * Hq * D / 81920.0) > 128 * 4096:
            hi, B = max(1, hi * 3 // 4), max(1, B * 3 // 4)
            if hi == 1 and B == 1:
                break
        return {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "ctx_lo": rng.randint(0, hi), "ctx_hi": hi,
                "nodes": nodes, "ragged": rng.random() < 0.6, "bs": rng.choice([16, 16, 16, 16, 32, 64, 8, 4]),
                "dtype": dtype}
    nodes = _spread(rng, 1, 61)
    layers = rng.choice([2, 24, 36, 48, 64])
    B = _spread(rng, 1, max(1, min(128, 32 * 61 * 64 * 1024 // (max(nodes, 16) * layers * Hkv * D))))
    hi = _spread(rng, 1, 4096)
    return {"op": op, "B": B, "layers": layers, "Hkv": Hkv, "D": D, "ctx_lo": rng.randint(0, hi), "ctx_hi": hi,
            "nodes": nodes, "accepted": rng.randint(1, max(1, min(8, (nodes + 1) // 2))),
            "bs": rng.choice([16, 16, 16, 32, 64, 8, 4]), "dtype": dtype}


# ------------------------------------------------------------------ sizes --

def _sizes(case):
    """(seq_lens, q_lens) of a case: fixed by the case, whatever the seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    B = case["B"]
    seq = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(B)]
    q = []
    for _ in range(B):
        n = case["nodes"]
        if case["op"] == "tables":
            if case["tree"]:
                n = r.randint(0, n)  # 0: a request that waits this step
            elif case["chunk"] and r.random() < 0.05:
                n = r.randint(1, case["chunk"])
        elif case["op"] == "attn" and case["ragged"]:
            n = r.randint(1, n)
        q.append(n)
    if sum(q) == 0:
        q[0] = 1
    return seq, q


def _kept(case, q):
    """How many nodes of each request's tree the model agrees with."""
    return [min(case["accepted"], (n + 1) // 2) for n in q]


def _blocks(n, bs):
    return (n + bs - 1) // bs


def _pad_rows(case):
    """Rows of the step behind the last request (a step padded to a fixed size)."""
    return 3 if case["op"] == "tables" and case["tree"] else 0


# ----------------------------------------------------------------- inputs --

def _random_tree(g, n):
    """A drafted tree: every node but the first hangs on an earlier one, more often on a recent one."""
    back = (g.random(n) ** 2 * np.arange(n)).astype(np.int64)
    parent = np.arange(n) - 1 - back
    parent[:1] = -1
    return parent


def _accepted_tree(g, n, keep):
    """A tree and the path of it that will be accepted. The path's nodes lie behind the places that they
    move to, so that a pass repeated on the same cache finds the same rows."""
    parent = _random_tree(g, n)
    path = [0] + sorted(int(x) for x in g.choice(np.arange(keep, n), size=keep - 1, replace=False)) if keep > 1 else [0]
    for a, b in zip(path, path[1:]):
        parent[b] = a
    return parent, path


def _mask_words(parent, words):
    rows = np.zeros((len(parent), words), np.uint64)
    for i, p in enumerate(parent):
        if p >= 0:
            rows[i] = rows[p]
        rows[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return rows.view(np.int64)


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(np.asarray(a, np.int32)), device=DEV)


def _cu(q):
    return np.concatenate([[0], np.cumsum(q)])


def prepare(case, seed):
    g = np.random.default_rng([seed, 7])
    tg = torch.Generator(device=DEV)
    tg.manual_seed(seed)
    seq, q = _sizes(case)
    B, bs = case["B"], case["bs"]
    T = int(sum(q))
    s = {"op": case["op"], "bs": bs, "B": B, "seq_lens": _i32(seq), "max_q": max(1, max(q))}
    if case["op"] == "tables":
        need = [_blocks(a + b, bs) for a, b in zip(seq, q)]
        held = [0 if case["fresh"] else _blocks(a, bs) for a in seq]
        width = max(case["width"], max(need))
        total = sum(max(n, h) for n, h in zip(need, held))
        num_blocks = total + 11
        perm = g.permutation(num_blocks)
        tab = np.full((B, width), -1, np.int32)
        at = 0
        for b, h in enumerate(held):
            tab[b, :h] = perm[at:at + h]
            at += h
        s.update(q_lens=_i32(q), tables=_i32(tab), held=_i32(held), free=_i32(perm[at:]), num_blocks=num_blocks,
                 total=T + _pad_rows(case), parents=None, no_mask=torch.zeros(0, dtype=torch.long, device=DEV))
        if case["tree"]:
            par = np.full(s["total"], -1, np.int32)
            cu = _cu(q)
            for b, n in enumerate(q):
                par[cu[b]:cu[b] + n] = _random_tree(g, n)
            s["parents"] = _i32(par)
        return s
    dtype = DTYPES[case["dtype"]]
    cu = _cu(q)
    words = (max(q) + 63) // 64
    if case["op"] == "attn":
        need = [_blocks(a + b, bs) for a, b in zip(seq, q)]
        num_blocks = sum(need) + 3
        perm = g.permutation(num_blocks)
        tab = np.full((B, max(need)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            tab[b, :n] = perm[at:at + n]
            at += n
        mask = np.concatenate([_mask_words(_random_tree(g, n), words) for n in q])
        shape = (num_blocks, bs, case["Hkv"], case["D"])
        s.update(q=torch.randn(T, case["Hq"], case["D"], device=DEV, generator=tg).to(dtype),
                 k=torch.randn(shape, device=DEV, generator=tg, dtype=dtype),
                 v=torch.randn(shape, device=DEV, generator=tg, dtype=dtype), tables=_i32(tab), cu_q=_i32(cu),
                 mask=torch.as_tensor(mask, device=DEV), max_ctx=max(a + b for a, b in zip(seq, q)),
                 seq_host=seq, q_host=q)
        if own:
            from pageserve_b200.paged_attention import AttentionWorkspace
            s["workspace"] = AttentionWorkspace()
        return s
    # accept: the requests share the blocks of a common prefix and own the ones their new tokens fall into
    first = [a // bs for a in seq]
    need = [_blocks(a + b, bs) for a, b in zip(seq, q)]
    shared = max(first)
    num_blocks = shared + sum(n - f for n, f in zip(need, first)) + 1
    perm = g.permutation(num_blocks)
    tab = np.full((B, max(need)), -1, np.int32)
    at = shared
    masks, tokens, targets = [], g.integers(0, VOCAB, T), g.integers(0, VOCAB, T)
    for b, n in enumerate(q):
        tab[b, :first[b]] = perm[:first[b]]
        own_blocks = need[b] - first[b]
        tab[b, first[b]:need[b]] = perm[at:at + own_blocks]
        at += own_blocks
        parent, path = _accepted_tree(g, n, _kept(case, q)[b])
        masks.append(_mask_words(parent, words))
        for x, y in zip(path, path[1:]):
            tokens[cu[b] + y] = targets[cu[b] + x]
    shape = (case["layers"], num_blocks, bs, case["Hkv"], case["D"])
    s.update(tokens=torch.as_tensor(tokens, device=DEV), targets=_i32(targets), cu_q=_i32(cu), tables=_i32(tab),
             mask=torch.as_tensor(np.concatenate(masks), device=DEV), q_host=q, seq_host=seq,
             k=torch.randn(shape, device=DEV, generator=tg, dtype=dtype),
             v=torch.randn(shape, device=DEV, generator=tg, dtype=dtype))
    return s


# ------------------------------------------------------------ plain forms --

def _plain_tables(s):
    bs, T, B = s["bs"], s["total"], s["B"]
    seq, q, held, tab = s["seq_lens"].long(), s["q_lens"].long(), s["held"].long(), s["tables"]
    width = tab.shape[1]
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=tab.device), q.cumsum(0)])
    need = (seq + q + bs - 1) // bs
    take = (need - held).clamp_min(0)
    first = take.cumsum(0) - take
    col = torch.arange(width, device=tab.device)
    new = first[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    free = s["free"][new.clamp(0, s["free"].numel() - 1)]
    out = torch.where(col < held[:, None], tab, torch.where(fresh, free, torch.full_like(free, -1)))
    row = torch.arange(T, device=tab.device)
    b = (torch.searchsorted(cu, row, right=True) - 1).clamp(0, B - 1)
    inside = row < cu[-1]
    i = row - cu[b]
    at = torch.where(inside, seq[b] + i, 0)
    phys = out[b, at // bs].long()
    slots = torch.where(inside, phys * bs + at % bs, -1)
    if s["parents"] is None:
        mask, pos = torch.zeros(0, dtype=torch.long, device=tab.device), at
    else:
        words = (s["max_q"] + 63) // 64
        w = torch.arange(words, device=tab.device)
        mask = torch.zeros(T, words, dtype=torch.long, device=tab.device)
        depth = torch.full((T,), -1, dtype=torch.long, device=tab.device)
        parent = s["parents"].long()
        live = inside.clone()
        cur = i.clone()
        for _ in range(s["max_q"]):  # one generation of ancestors at a time
            bit = torch.ones_like(cur) << (cur.clamp_min(0) % 64)
            mask |= torch.where(live[:, None] & (w == (cur // 64)[:, None]), bit[:, None], 0)
            depth += live
            nxt = parent[(cu[b] + cur).clamp(0, T - 1)]
            live = live & (nxt >= 0)
            cur = torch.where(live, nxt, cur)
        pos = torch.where(inside, seq[b] + depth, 0)
    return (out, torch.maximum(held, need).int(), cu.int(), pos.int(), slots.int(), mask, take.sum().int().reshape(1))


def _plain_attn(s):
    q, k, v, bs = s["q"], s["k"], s["v"], s["bs"]
    hq, d = q.shape[1:]
    hkv = k.shape[2]
    out = torch.empty_like(q)
    fk, fv = k.reshape(-1, hkv, d), v.reshape(-1, hkv, d)
    bit = torch.arange(s["max_q"], device=q.device)
    at = 0
    for b, (n0, n) in enumerate(zip(s["seq_host"], s["q_host"])):
        pos = torch.arange(n0 + n, device=q.device)
        slot = s["tables"][b].long()[pos // bs] * bs + pos % bs
        kb = fk[slot].float().permute(1, 2, 0)  # hkv, d, keys
        vb = fv[slot].float().permute(1, 0, 2)  # hkv, keys, d
        qb = q[at:at + n].float().reshape(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        sc = torch.matmul(qb * (1.0 / math.sqrt(d)), kb).reshape(hkv, hq // hkv, n, n0 + n)
        words = s["mask"][at:at + n]
        sees = (words[:, bit[:n] // 64] >> (bit[:n] % 64) & 1) != 0
        sc[..., n0:] = torch.where(sees, sc[..., n0:], -math.inf)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        o = torch.matmul(p.reshape(hkv, -1, n0 + n), vb).reshape(hkv, hq // hkv, n, d)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(q.dtype)
        at += n
    return out


def _plain_accept(s):
    bs, B, limit = s["bs"], s["B"], s["max_q"]
    dev = s["tokens"].device
    num = torch.zeros(B, dtype=torch.int32, device=dev)
    nodes = torch.full((B, limit), -1, dtype=torch.int32, device=dev)
    toks = torch.full((B, limit), -1, dtype=torch.int32, device=dev)
    src, dst = [], []
    bit = torch.arange(limit, device=dev)
    at = 0
    for b, n in enumerate(s["q_host"]):
        words = s["mask"][at:at + n]
        up = (words[:, bit[:n] // 64] >> (bit[:n] % 64) & 1) != 0  # node, its ancestors and itself
        i = bit[:n]
        parent = torch.where(up & (i < i[:, None]), i, -1).amax(1)
        tok, tgt = s["tokens"][at:at + n], s["targets"][at:at + n].long()
        agrees = ((parent >= 0) & (tok == tgt[parent.clamp_min(0)])) | (i == 0)
        whole = (agrees | ~up).all(1)
        depth = torch.where(whole, up.sum(1), 0)
        best = torch.argmax(depth * n + (n - 1 - i))  # the deepest, the lowest of them
        path = torch.nonzero(up[best]).flatten()
        m = path.numel()
        num[b] = m
        nodes[b, :m] = path.int()
        toks[b, :m] = tgt[path].int()
        row = s["tables"][b].long()
        a, c = s["seq_lens"][b].long() + path, s["seq_lens"][b].long() + bit[:m]
        src.append(row[a // bs] * bs + a % bs)
        dst.append(row[c // bs] * bs + c % bs)
        at += n
    src, dst = torch.cat(src), torch.cat(dst)
    for c in (s["k"], s["v"]):
        flat = c.view(c.shape[0], -1, *c.shape[3:])
        flat[:, dst] = flat[:, src]
    return num, nodes, toks, s["seq_lens"] + num, s["k"], s["v"]


# -------------------------------------------------------------------- run --

def run(s):
    if not own:
        return {"tables": _plain_tables, "attn": _plain_attn, "accept": _plain_accept}[s["op"]](s)
    from pageserve_b200 import speculative
    if s["op"] == "tables":
        r = speculative.build_step_tables(s["seq_lens"], s["q_lens"], s["tables"], s["held"], s["free"],
                                          s["num_blocks"], s["bs"], s["total"], parents=s["parents"],
                                          max_q_len=s["max_q"])
        mask = r.tree_mask if r.tree_mask is not None else s["no_mask"]
        return r.block_tables, r.held, r.cu_q, r.positions, r.slots, mask, r.free_used
    if s["op"] == "attn":
        return speculative.tree_attention(s["q"], s["k"], s["v"], s["tables"], s["cu_q"], s["seq_lens"], s["mask"],
                                          s["max_q"], s["max_ctx"], workspace=s["workspace"])
    a = speculative.accept_trees(s["tokens"], s["targets"], s["mask"], s["cu_q"], s["seq_lens"], s["max_q"], s["k"],
                                 s["v"], s["tables"])
    return a.num, a.nodes, a.tokens, a.start_pos, s["k"], s["v"]


# ------------------------------------------------------------------- work --

def work(case):
    seq, q = _sizes(case)
    T, B, bs = sum(q), case["B"], case["bs"]
    if case["op"] == "tables":
        need = [_blocks(a + b, bs) for a, b in zip(seq, q)]
        held = [0 if case["fresh"] else _blocks(a, bs) for a in seq]
        width = max(case["width"], max(need))
        rows = T + _pad_rows(case)
        words = (max(1, max(q)) + 63) // 64
        read = 12 * B + 4 * sum(held) + 4 * sum(max(0, n - h) for n, h in zip(need, held))
        write = 4 * B * width + 4 * B + 4 * (B + 1) + 8 * rows + 4
        if case["tree"]:
            read += 4 * rows
            write += 8 * rows * words
        return {"bytes": read + write, "flops": 0}
    if case["op"] == "attn":
        words = (max(q) + 63) // 64
        keys = sum(a + b for a, b in zip(seq, q))
        io = 2 * 2 * T * case["Hq"] * case["D"]
        cache = 2 * 2 * keys * case["Hkv"] * case["D"]
        meta = 4 * sum(_blocks(a + b, bs) for a, b in zip(seq, q)) + 8 * T * words + 8 * B
        # a node sees its context and, at the least, itself
        return {"bytes": io + cache + meta, "flops": 4 * case["Hq"] * case["D"] * sum(b * (a + 1) for a, b in zip(seq, q))}
    words = (max(q) + 63) // 64
    kept = _kept(case, q)
    moved = sum(k - 1 for k in kept) * 2 * 2 * case["layers"] * case["Hkv"] * case["D"]
    return {"bytes": 2 * moved + T * (8 + 4 + 8 * words) + 12 * B + 8 * B * max(q), "flops": 0}


# ------------------------------------------------------------------ exact --

def _ancestors(row):
    """The nodes that a mask row names, ascending."""
    return [64 * w + j for w, x in enumerate(row) for j in range(64) if (x >> j) & 1]


def exact(case, seed):
    s = prepare(case, seed)
    bs, B = case["bs"], case["B"]
    seq, q = _sizes(case)
    cu = _cu(q).tolist()
    if case["op"] == "tables":
        tab, held, free = s["tables"].tolist(), s["held"].tolist(), s["free"].tolist()
        used, pos, slots, masks = 0, [], [], []
        words = (s["max_q"] + 63) // 64
        par = s["parents"].tolist() if s["parents"] is not None else None
        for b in range(B):
            row, n = tab[b], held[b]
            while n * bs < seq[b] + q[b]:
                row[n] = free[used]
                used, n = used + 1, n + 1
            held[b] = n
            for j in range(n, len(row)):
                row[j] = -1
            up = []
            for i in range(q[b]):
                p = seq[b] + i
                slots.append(row[p // bs] * bs + p % bs)
                if par is None:
                    pos.append(p)
                else:
                    m = par[cu[b] + i]
                    up.append((up[m] if m >= 0 else 0) | 1 << i)
                    pos.append(seq[b] + bin(up[-1]).count("1") - 1)
            masks += up
        pad = s["total"] - len(pos)
        pos, slots = pos + [0] * pad, slots + [-1] * pad
        if par is None:
            mask = torch.zeros(0, dtype=torch.long)
        else:
            rows = [[(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for m in masks + [0] * pad]
            mask = torch.from_numpy(np.asarray(rows, np.uint64).view(np.int64))
        t = [torch.tensor(tab), torch.tensor(held), torch.tensor(cu), torch.tensor(pos), torch.tensor(slots)]
        return tuple(x.int().to(DEV) for x in t) + (mask.to(DEV), torch.tensor([used], dtype=torch.int32, device=DEV))
    rows = s["mask"].tolist()
    up = [_ancestors([x & (2 ** 64 - 1) for x in r]) for r in rows]
    if case["op"] == "attn":
        hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
        out = torch.zeros(sum(q), hq, d, dtype=torch.float64, device=DEV)
        for b in range(B):
            n0, n = seq[b], q[b]
            blocks = s["tables"][b, :_blocks(n0 + n, bs)].long()
            kb = s["k"][blocks].reshape(-1, hkv, d)[:n0 + n].double()
            vb = s["v"][blocks].reshape(-1, hkv, d)[:n0 + n].double()
            sees = torch.zeros(n, n0 + n, dtype=torch.bool)
            sees[:, :n0] = True
            for i in range(n):
                sees[i, [n0 + j for j in up[cu[b] + i]]] = True
            sees = sees.to(DEV)
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                qb = s["q"][cu[b]:cu[b + 1], heads].double()
                sc = torch.einsum("ngd,kd->ngk", qb, kb[:, h]) / math.sqrt(d)
                w = torch.softmax(sc.masked_fill(~sees[:, None, :], -math.inf), -1)
                out[cu[b]:cu[b + 1], heads] = torch.einsum("ngk,kd->ngd", w, vb[:, h])
        return out
    tok, tgt, tab = s["tokens"].tolist(), s["targets"].tolist(), s["tables"].tolist()
    limit = s["max_q"]
    num, nodes, toks, start = [], [], [], []
    old_k, old_v = s["k"].clone(), s["v"].clone()
    src, dst = [], []
    for b in range(B):
        good = {0: [0]}
        for i in range(1, q[b]):
            line = up[cu[b] + i]
            if len(line) > 1 and line[-2] in good and tok[cu[b] + i] == tgt[cu[b] + line[-2]]:
                good[i] = good[line[-2]] + [i]
        path = max(good.values(), key=lambda p: (len(p), -p[-1]))
        num.append(len(path))
        nodes.append(path + [-1] * (limit - len(path)))
        toks.append([tgt[cu[b] + x] for x in path] + [-1] * (limit - len(path)))
        start.append(seq[b] + len(path))
        for j, x in enumerate(path):
            src.append((tab[b][(seq[b] + x) // bs], (seq[b] + x) % bs))
            dst.append((tab[b][(seq[b] + j) // bs], (seq[b] + j) % bs))
    (sb, so), (db, do) = torch.tensor(src, device=DEV).T, torch.tensor(dst, device=DEV).T
    s["k"][:, db, do] = old_k[:, sb, so]
    s["v"][:, db, do] = old_v[:, sb, so]
    return (_i32(num), _i32(nodes), _i32(toks), _i32(start), s["k"], s["v"])
