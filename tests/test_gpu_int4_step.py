"""The step of a 4-bit group that ends at fp16's largest value, bit for bit, on an MI355X:
the next smaller one is taken where m + 15 s would round to infinity, and nowhere else."""

from __future__ import annotations

import numpy as np
import pytest

from tests import int4_ref as ref

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def groups(lows, highs):
    """Rows [n, 128] whose groups span every pair of a low and a high, in between values
    spread over the pair's range."""
    pairs = np.array([(a, b) for a in lows for b in highs if a <= b])
    pairs = np.concatenate((pairs, np.repeat(pairs[-1:], -len(pairs) % 4, 0)))
    x = pairs[:, :1] + (pairs[:, 1:] - pairs[:, :1]) * np.linspace(0, 1, 32)[None]
    x = x.astype(np.float16)
    x[:, 0], x[:, 31] = pairs[:, 0], pairs[:, 1]
    x = x[:, np.random.default_rng(1).permutation(32)]
    return x.reshape(-1, 128)


HALVES = np.arange(65536, dtype=np.uint16).view(np.float16)
HIGHS = HALVES[np.isfinite(HALVES) & (HALVES >= 65000)].astype(np.float64)


@pytest.mark.parametrize("lows", [
    -(2.0 ** -np.arange(0, 25)), 2.0 ** -np.arange(0, 25), np.linspace(-0.01, 0.01, 401),
    HALVES[np.isfinite(HALVES)][::61].astype(np.float64), [0.0, -0.0, 60000, 65472, 65504, -65504]],
    ids=["below 0", "over 0", "around 0", "all", "ends"])
def test_the_step_at_the_end_of_fp16(lows):
    from latentserve_amd.kernels.hip import int4_cache as i4

    x = groups(np.asarray(lows, np.float64).astype(np.float16).astype(np.float64), HIGHS)
    n = len(x)
    nb = -(-n // 16)
    print(f"step groups={4 * n}", flush=True)
    pools = i4.empty_pools(nb, 1, "cuda")
    rows = torch.from_numpy(x).cuda().view(1, 1, n, 128)
    i4.write(rows, rows, torch.arange(n, device="cuda"), pools)
    codes, s, m = ref.quantize(x)
    kc, ka, vc, va = (p.cpu().numpy() for p in pools)
    tok = np.arange(n)
    blk, t = tok // 16, tok % 16
    np.testing.assert_array_equal(ka[blk, 0, t, :, 0], s)
    np.testing.assert_array_equal(va[blk, 0, :, t // 4, 0, t % 4], s)
    table = torch.arange(nb, device="cuda").int()[None]
    for got in i4.read(pools, table, torch.tensor([n], device="cuda").int(), n):
        got = got.cpu().numpy()[0, 0]
        assert np.isfinite(got).all()
        np.testing.assert_array_equal(got, ref.values(codes, s, m))
