"""The weights of 4-bit decode attention hold fp32's accuracy, on an MI355X.

Queries with one channel of 1 make the scores single entries of K, exact in fp32, so what
is off comes from the weights and the sums alone.  Bounds, of the weights' mean of |v|
(`mag`), the largest weight 1:

  exponent   its argument, below 32 in log2 units, rounds twice (2^-24 of 32 each, 2^-18 ln 2
             of a weight), the exponential by 2^-22; numerator and denominator: 2^-17 in all
  weights    21 bits and more, and no less than 2^-39 of the largest one: 2^-20, and 2^-39
             a token
  sums       a wave's steps of 32 tokens, its merges: below 2^11 additions of 2^-24, as often
             as not of either sign: 2^-17
  result     half a step of fp16"""

from __future__ import annotations

import numpy as np
import pytest

from tests import int4_ref as ref

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def attend(q, arrays, tables, lens, scale):
    from latentserve_amd.kernels.hip import int4_cache as i4
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    out = i4.paged_decode_int4(dev(q), i4.Int4Pools(*(dev(a) for a in arrays)), dev(tables),
                               dev(lens), softmax_scale=scale)
    return out.cpu().numpy()


def half_step(want):
    return np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2


def one_hot(b, h, r):
    """[b, h, r, 128], row i of a head the channel 37 i + 11 h + 5 b."""
    q = np.zeros((b, h, r, 128), np.float16)
    for i in range(b):
        for j in range(h):
            for k in range(r):
                q[i, j, k, (37 * k + 11 * j + 5 * i) % 128] = 1
    return q


@pytest.mark.parametrize("signs", ["positive", "both"])
@pytest.mark.parametrize("lens,h,r", [([2, 3, 5, 8, 17, 33, 1], 2, 6), ([300, 47, 1000], 2, 6),
                                      ([300, 2, 1000], 1, 8), ([300, 2, 1000], 2, 9),
                                      ([129, 40], 3, 16), ([700, 31], 1, 1), ([20000], 2, 6)],
                         ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_results_are_off_by_a_rounding_of_the_result(lens, h, r, signs):
    """Of sums of both signs a result is small against its terms, and the weights' roundings
    show."""
    width, nb = -(-max(lens) // 16), 40
    arrays = ref.random_pools(nb, h, 3)
    # entries of K 0 .. 7.5, of V 1 .. 1.94 or -0.94 .. 0.94
    arrays[1][..., 0], arrays[1][..., 1] = 0.5, 0
    aff = arrays[3].reshape(nb, h, 4, 4, 2, 4)
    aff[..., 0, :], aff[..., 1, :] = (0.0625, 1) if signs == "positive" else (0.125, -0.9375)
    tables = np.random.default_rng(4).integers(0, nb, (len(lens), width)).astype(np.int32)
    q, scale = one_hot(len(lens), h, r), 1.0
    print(f"weights lens={lens} h={h} r={r}", flush=True)
    got = attend(q, arrays, tables, np.array(lens, np.int32), scale).astype(np.float64)
    kv, vv = (ref.pool_values(arrays[2 * z], arrays[2 * z + 1], z == 1).astype(np.float64)
              for z in (0, 1))
    for i, n in enumerate(lens):
        pos = np.arange(n)
        blk, t = tables[i, pos // 16], pos % 16
        for j in range(h):
            x = q[i, j].astype(np.float64) @ kv[blk, j, t].T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            z = p.sum(-1, keepdims=True)
            want, mag = p @ vv[blk, j, t] / z, p @ np.abs(vv[blk, j, t]) / z
            tol = half_step(want) + mag * (2.0 ** -16 + 2.0 ** -20) + n * 2.0 ** -39 * 2 / z
            bad = np.abs(got[i, j] - want) > tol
            assert not bad.any(), (n, j, bad.sum(), (np.abs(got[i, j] - want) - tol).max())


@pytest.mark.parametrize("gap", [4.0, 10.0, 16.0, 17.5, 20.0, 23.0])
@pytest.mark.parametrize("at", ["first", "last", "none"])
@pytest.mark.parametrize("n,h,r", [(100003, 1, 2), (6400, 520, 2), (6400, 520, 16)])
def test_a_long_tail_under_one_large_score_keeps_its_mass(n, h, r, at, gap):
    """One token `gap` nats over many even ones, its value 0 and theirs 1: the result is the
    tail's share.  (520 heads: a workgroup each, whose four waves walk the sequence.)"""
    pages = -(-n // 16)
    # block 0: the tail; block 1: the same with the large score at token 3
    arrays = ref.random_pools(2, h, 5)
    for a in arrays:
        a[...] = 0
    arrays[1][..., 0] = 1                                    # K: entry = code
    vaff = arrays[3].reshape(2, h, 4, 4, 2, 4)
    vaff[..., 1, :] = 1                                      # V: 1
    byte, shift = ref.code_at(11, False, 3)
    arrays[0][1].reshape(h, -1)[:, byte] = 8 << shift
    vaff[1, :, :, 0, 1, 3] = 0
    tables = np.zeros((1, pages), np.int32)
    if at != "none":
        tables[0, 0 if at == "first" else pages - 2] = 1
    q = np.zeros((1, h, r, 128), np.float16)
    q[..., 11] = 1
    print(f"tail n={n} h={h} r={r} gap={gap} {at}", flush=True)
    got = attend(q, arrays, tables, np.array([n], np.int32), gap / 8).astype(np.float64)
    tail = (n - 1) * np.exp(-gap)
    want = 1.0 if at == "none" else tail / (1 + tail)
    tol = half_step(np.array(want)) + want * (2.0 ** -16 + 2.0 ** -20) + n * 2.0 ** -39 / (1 + tail)
    assert (np.abs(got - want) <= tol).all(), (got.min(), got.max(), want, tol)


def test_scores_far_past_fp16_give_finite_results():
    """q and k of 30000 and more: scores of 10^10, whose rounding in fp32 is thousands.
    A sequence of equal ones is their mean."""
    h, r = 1, 3
    arrays = ref.random_pools(2, h, 7)
    arrays[0][...] = 0
    arrays[1][..., 0], arrays[1][..., 1] = 0, 30000
    vv = ref.pool_values(arrays[2], arrays[3], True).astype(np.float64)
    tables, lens = np.array([[0, 1], [1, 0]], np.int32), np.array([32, 1], np.int32)
    for size in (1.0, 64.0, 1024.0):
        q = np.full((2, h, r, 128), size, np.float16)
        got = attend(q, arrays, tables, lens, 0.088).astype(np.float64)
        mean = vv[:, 0].reshape(32, 128).mean(0)
        mag = np.abs(vv[:, 0]).reshape(32, 128).mean(0)
        assert np.isfinite(got).all(), size
        assert (np.abs(got[0] - mean) <= half_step(mean) + mag * 2.0 ** -16).all(), size
        assert (np.abs(got[1] - vv[1, 0, 0]) <= half_step(vv[1, 0, 0])
                + np.abs(vv[1, 0, 0]) * 2.0 ** -16).all(), size
