"""What the drafted-tree and eviction operators compute, in numpy and 64 bits, from their
definitions, with bounds on what 32-bit sums and fp16 weights may add."""

from __future__ import annotations

import numpy as np

HALF = 2.0 ** -11                       # half a step of fp16, relative
SINGLE = 2.0 ** -24


def random_tree(n, rng, roots=1):
    """Parents of a random tree: the first `roots` nodes have none."""
    return np.array([-1 if i < roots else int(rng.integers(0, i)) for i in range(n)], np.int32)


def seen_by(parents):
    """bool [N, N]: row i, column j: node i sees node j."""
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i in range(n):
        at = i
        while at >= 0:
            m[i, at] = True
            up = parents[at]
            at = up if 0 <= up < at else -1
    return m


def words_of(seen):
    """bool [..., N, N] -> int64 mask words [..., N, words]."""
    n = seen.shape[-1]
    out = np.zeros(seen.shape[:-1] + (-(-n // 64),), np.uint64)
    for j in range(n):
        out[..., j // 64] |= seen[..., j].astype(np.uint64) << np.uint64(j % 64)
    return out.view(np.int64)


def rows_of(pool, table, length):
    """(rows [length, H, 128] fp64, exists [length]) of a sequence's tokens."""
    nb = pool.shape[0]
    pos = np.arange(length)
    inside = pos < len(table) * 16
    blk = np.where(inside, table[np.minimum(pos // 16, len(table) - 1)], -1)
    ok = (blk >= 0) & (blk < nb)
    out = pool[np.where(ok, blk, 0), pos % 16].astype(np.float64)
    out[~ok] = 0
    return out, ok


def attend(q, k_pool, v_pool, tables, lens, seen=None, counts=None, scale=128.0 ** -0.5):
    """q [B, N, H, r, 128] -> out, lse, the bound on out's error, the bound on lse's.
    seen [B, N, N] bool (None: a chain)."""
    b, n, h, r, d = q.shape
    out = np.zeros(q.shape)
    lse = np.full((b, n, h, r), -np.inf)
    tol, ltol = np.zeros(q.shape), np.zeros((b, n, h, r))
    for s in range(b):
        length = max(0, int(lens[s]))
        ctx = max(0, length - n)
        nodes = min(length, n if counts is None else min(n, max(0, int(counts[s]))))
        k, ok = rows_of(k_pool, tables[s], length)
        v, _ = rows_of(v_pool, tables[s], length)
        for i in range(nodes):
            see = np.zeros(length, bool)
            see[:ctx] = True
            row = np.arange(n) <= i if seen is None else seen[s, i]
            see[ctx:ctx + nodes] = row[:nodes]
            see &= ok
            if not see.any():
                continue
            ks, vs = k[see], v[see]
            for hh in range(h):
                x = q[s, i, hh].astype(np.float64) @ ks[:, hh].T * scale          # [r, t]
                size = np.abs(q[s, i, hh].astype(np.float64)) @ np.abs(ks[:, hh]).T * scale
                top = x.max(-1, keepdims=True)
                e = np.exp(x - top)
                z = e.sum(-1, keepdims=True)
                p = e / z
                out[s, i, hh] = p @ vs[:, hh]
                lse[s, i, hh] = (top + np.log(z))[:, 0]
                # a score: 128 products summed in 32 bits; the exponent's scale and
                # subtraction (log2 units); 2^x to 2^-22
                ds = (136 * SINGLE * size.max(-1) + 4 * SINGLE * np.abs(x).max(-1) + 2.0 ** -21)
                mass = p @ np.abs(vs[:, hh])
                t = int(see.sum())
                # weights rounded to fp16 (half a step each; below 2^-21 of the largest an
                # absolute 2^-32 of it), 32-bit sums, the result's own rounding
                tol[s, i, hh] = mass * HALF + (mass + np.abs(out[s, i, hh])) * (2 * ds[:, None] + t * SINGLE) \
                    + t * 2.0 ** -31 * np.abs(vs[:, hh]).max(0) + HALF * np.abs(out[s, i, hh]) + 2.0 ** -24
                # (of the weights before they are rounded)
                ltol[s, i, hh] = 2 * ds + t * SINGLE + 2.0 ** -20 + 3 * SINGLE * np.abs(lse[s, i, hh])
    return out, lse, tol, ltol


def path_weights(q, lse, k_pool, tables, lens, path, lengths, scale=128.0 ** -0.5):
    """What add_weights adds: [B, H, T], and the bound on its error (T: the longest)."""
    b, n, h, r, d = q.shape
    most = max(int(max(lens)), 1)
    add, tol = np.zeros((b, h, most)), np.zeros((b, h, most))
    for s in range(b):
        length = max(0, int(lens[s]))
        count = min(length, max(0, int(lengths[s])))
        k, ok = rows_of(k_pool, tables[s], length)
        for i in range(count):
            node = int(path[s, i])
            if not 0 <= node < n:
                continue
            end = length - count + i + 1
            for hh in range(h):
                qq = q[s, node, hh].astype(np.float64)
                x = qq @ k[:end, hh].T * scale
                size = np.abs(qq) @ np.abs(k[:end, hh]).T * scale
                for rr in range(r):
                    ls = float(lse[s, node, hh, rr])
                    if ls == -np.inf:
                        continue
                    p = np.where(ok[:end], np.exp(x[rr] - ls), 0)
                    add[s, hh, :end] += p
                    # the score, the statistic in log2 units, 2^x, the sum over rows
                    tol[s, hh, :end] += p * (136 * SINGLE * size[rr] + 6 * SINGLE *
                                             (np.abs(x[rr]) + abs(ls)) * 1.5 + 2.0 ** -21
                                             + count * r * SINGLE)
    return add, tol


def accepted(tokens, parents, choices, nodes):
    """(path, next token) of one tree."""
    if nodes <= 0:
        return [], -1
    at, path = 0, [0]
    while True:
        child = [j for j in range(at + 1, nodes) if parents[j] == at and tokens[j] == choices[at]]
        if not child:
            return path, int(choices[at])
        at = child[0]
        path.append(at)


def selected(sums, length, budget, sinks, recent):
    """Positions kept of one row."""
    length = max(0, min(int(length), len(sums)))
    if length <= budget:
        return list(range(length))
    forced = [t for t in range(length) if t < sinks or t >= length - recent]
    others = [t for t in range(length) if sinks <= t < length - recent]
    others.sort(key=lambda t: (0, 0.0, t) if np.isnan(sums[t]) else (1, -float(sums[t]), t))
    return sorted(forced + others[:budget - len(forced)])
