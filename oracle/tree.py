"""numpy restatement, in 64 bits, of the operators of decoding with drafted
token trees: the step's tables, the tree attention and the acceptance. Written
from the definitions (sets of ancestors, one key at a time), without masks as
bit words and without the package's code."""

from __future__ import annotations

import numpy as np


def ancestors(parents) -> list[set[int]]:
    """Node -> the set of its ancestors and itself; parents outside [-1, i)
    count as none."""
    out: list[set[int]] = []
    for i, p in enumerate(parents):
        out.append(({i} | out[p]) if 0 <= p < i else {i})
    return out


def mask_words(sets, words: int) -> np.ndarray:
    """Sets of nodes -> int64 bit words (node j is bit j % 64 of word j // 64)."""
    rows = [[sum(1 << (j - 64 * w) for j in s if j // 64 == w) for w in range(words)] for s in sets]
    return np.asarray(rows, np.uint64).reshape(len(rows), words).view(np.int64)


def word_sets(mask: np.ndarray) -> list[set[int]]:
    return [{64 * w + j for w, x in enumerate(row) for j in range(64) if (int(x) >> j) & 1}
            for row in np.asarray(mask).view(np.uint64)]


def step_tables(seq_lens, q_lens, tables, held, free, block_size, total, parents=None, max_q_len=0):
    """(tables, held, cu_q, positions, slots, mask, free_used) of a step whose
    lengths, parents and free list are in order."""
    tables = np.array(tables, np.int64)
    held = list(map(int, held))
    free = list(map(int, free))
    used, cu, pos, slots, sets = 0, [0], [], [], []
    for b, (n0, n) in enumerate(zip(seq_lens, q_lens)):
        while held[b] * block_size < n0 + n:
            tables[b, held[b]] = free[used]
            used += 1
            held[b] += 1
        tables[b, held[b]:] = -1
        up = None if parents is None else ancestors(parents[cu[-1]:cu[-1] + n])
        for i in range(n):
            at = n0 + i
            slots.append(int(tables[b, at // block_size]) * block_size + at % block_size)
            pos.append(at if up is None else n0 + len(up[i]) - 1)
        sets += up or []
        cu.append(cu[-1] + n)
    pad = total - len(pos)
    pos, slots = pos + [0] * pad, slots + [-1] * pad
    mask = None if parents is None else mask_words(sets + [set()] * pad, (max_q_len + 63) // 64)
    return tables, np.array(held), np.array(cu), np.array(pos), np.array(slots), mask, used


def tree_attention(q, k_cache, v_cache, tables, cu_q, start_pos, sets):
    """(out, bound) in 64 bits: out (T, Hq, D) and, for tolerances, the sum of
    weight times |v| behind each output value."""
    T, hq, d = q.shape
    bs, hkv = k_cache.shape[1:3]
    out = np.zeros((T, hq, d))
    mag = np.zeros((T, hq, d))
    for b in range(len(start_pos)):
        for i in range(cu_q[b + 1] - cu_q[b]):
            row = cu_q[b] + i
            keys = list(range(start_pos[b])) + [start_pos[b] + j for j in sorted(sets[row])
                                                if j < cu_q[b + 1] - cu_q[b]]
            if not keys:
                continue
            at = [(int(tables[b][p // bs]), p % bs) for p in keys]
            kk = np.stack([k_cache[x, y] for x, y in at]).astype(np.float64)
            vv = np.stack([v_cache[x, y] for x, y in at]).astype(np.float64)
            for h in range(hq):
                kv = h // (hq // hkv)
                s = kk[:, kv] @ q[row, h].astype(np.float64) / np.sqrt(d)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[row, h] = w @ vv[:, kv]
                mag[row, h] = w @ np.abs(vv[:, kv])
    return out, mag


def accept(tokens, targets, sets):
    """The accepted path of one tree (a list of its nodes)."""
    good = {}
    for i in range(len(tokens)):
        line = sorted(sets[i])
        if i == 0:
            good[0] = [0] if line == [0] else None
            continue
        above = [j for j in line if j < i]
        if above and good.get(above[-1]) and tokens[i] == targets[above[-1]] and line == good[above[-1]] + [i]:
            good[i] = line
    best = [p for p in good.values() if p]
    return max(best, key=lambda p: (len(p), -p[-1])) if best else [0]


def move_rows(cache, table, block_size, start, path):
    """cache (L, NB, bs, Hkv, D): the path's rows at start + node -> start + k
    (from a copy: no order of the moves matters)."""
    old = cache.copy()
    for k, j in enumerate(path):
        a, c = start + j, start + k
        cache[:, table[c // block_size], c % block_size] = old[:, table[a // block_size], a % block_size]
