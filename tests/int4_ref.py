"""The 4-bit cache in numpy and 64 bits, from its definition: no code shared with the
package."""

from __future__ import annotations

import math

import numpy as np


def quantize(x):
    """x [..., 128] fp16 -> codes [..., 128] int, s and m [..., 4] fp16."""
    g = x.reshape(x.shape[:-1] + (4, 32))
    lo, hi = g.min(-1), g.max(-1)
    s = ((hi.astype(np.float32) - lo.astype(np.float32)) / np.float32(15)).astype(np.float16)
    over = lo.astype(np.float64) + 15 * s.astype(np.float64) >= 65520      # rounds to inf
    s = np.where(over, np.nextafter(s, np.float16(0)), s)
    d = g.astype(np.float64) - lo.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.rint(d / s.astype(np.float64)[..., None])
    c = np.where(s[..., None] == 0, 0, np.clip(c, 0, 15)).astype(np.int64)
    return c.reshape(x.shape), s, lo


def values(codes, s, m):
    """fp16(m + s * code), rounded once."""
    g = codes.reshape(codes.shape[:-1] + (4, 32)).astype(np.float64)
    v = m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * g
    return v.astype(np.float16).reshape(codes.shape)


def code_at(c, value, t):
    """(byte of a (page, head)'s codes, shift) of channel c of token t."""
    if value:
        return 64 * (c // 8) + 4 * t + c % 8 // 2, 4 * (c % 2)
    return 64 * t + 16 * (c // 8 % 4) + 4 * (c // 32) + c % 8 // 2, 4 * (c % 2)


def affine_at(c, value, t):
    """Index of s (of m: the second) among a (page, head)'s 128 fp16."""
    if value:
        s = 32 * (c // 32) + 8 * (t // 4) + t % 4
        return s, s + 4
    s = 8 * t + 2 * (c // 32)
    return s, s + 1


def entry(codes, affine, value, blk, h, t):
    """Values [128] of one token: codes / affine numpy pools of any shape [nb, H, ...]."""
    raw, aff = codes[blk, h].reshape(-1), affine[blk, h].reshape(-1)
    out = np.empty(128, dtype=np.float16)
    for c in range(128):
        byte, shift = code_at(c, value, t)
        si, mi = affine_at(c, value, t)
        code = (int(raw[byte]) >> shift) & 15
        with np.errstate(invalid="ignore", over="ignore"):
            out[c] = np.float16(np.float64(aff[mi]) + np.float64(aff[si]) * code)
    return out


def pool_values(codes, affine, value):
    """[nb, H, 16, 128] fp16: every entry (entry(), all at once)."""
    nb, h = codes.shape[:2]
    raw, aff = codes.reshape(nb, h, -1), affine.reshape(nb, h, -1).astype(np.float64)
    c, t = np.arange(128)[None, :], np.arange(16)[:, None]
    byte, shift = np.vectorize(lambda a, b: code_at(a, value, b))(c, t)
    si, mi = np.vectorize(lambda a, b: affine_at(a, value, b))(c, t)
    code = (raw[:, :, byte].astype(np.int64) >> shift) & 15
    with np.errstate(invalid="ignore", over="ignore"):
        return (aff[:, :, mi] + aff[:, :, si] * code).astype(np.float16)


def random_pools(nb, heads, seed):
    """numpy pools with codes of all values and steps and minima around unit size."""
    r = np.random.default_rng(seed)
    ks = (0.15 + 0.25 * r.random((nb, heads, 16, 4))).astype(np.float16)
    vs = (0.15 + 0.25 * r.random((nb, heads, 4, 4, 4))).astype(np.float16)
    km = (-7.5 * ks + 0.3 * r.standard_normal(ks.shape)).astype(np.float16)
    vm = (-7.5 * vs + 0.3 * r.standard_normal(vs.shape)).astype(np.float16)
    return (r.integers(0, 256, (nb, heads, 16, 64), dtype=np.uint8), np.stack((ks, km), -1),
            r.integers(0, 256, (nb, heads, 16, 16, 4), dtype=np.uint8), np.stack((vs, vm), -2))


def attend(q, kv, vv, tables, lens, scale=None):
    """64-bit attention and a bound on the kernel's error: q [B, H, R, 128], kv / vv
    pool_values.  Blocks outside the pool are skipped.

    The bound, a half step u = 2^-11 of fp16: the weights p are rounded to fp16
    (u p each, and 2^-25 where p is subnormal, at most one a token), the result is
    (u |out|), and the scores, 128 fp32 products and sums, and the exponential are off
    by at most 256 * 2^-24 sum |q k| scale + 2^-20 relative in p, twice (numerator and
    denominator)."""
    b, h, r, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    nb, u = kv.shape[0], 2.0 ** -11
    for i in range(b):
        n = min(int(lens[i]), tables.shape[1] * 16)
        pos = np.arange(max(n, 0))
        blk = tables[i, pos // 16]
        ok = (blk >= 0) & (blk < nb)
        if not ok.any():
            continue
        blk, t = blk[ok], pos[ok] % 16
        for hh in range(h):
            k, v = (x[blk, hh, t].astype(np.float64) for x in (kv, vv))
            qq = q[i, hh].astype(np.float64)
            x = qq @ k.T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            z = p.sum(-1, keepdims=True)
            out[i, hh] = p @ v / z
            mag = p @ np.abs(v) / z
            ds = (np.abs(qq) @ np.abs(k).T * abs(scale)).max(-1, keepdims=True) * 256 * 2.0 ** -24
            tol[i, hh] = (u * (mag + np.abs(out[i, hh])) + 2 * mag * (ds + 2.0 ** -20)
                          + len(t) * 2.0 ** -25 * np.abs(v).max() / z + 2.0 ** -24)
    return out, tol
