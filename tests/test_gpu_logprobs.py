"""Token log probabilities against 64 bits, on an MI355X.

Bounds (u = 2^-24, half a step of fp32): an fp32 exp of |d| <= D is off by about (D + 4)
u relative (its argument's rounding), sums of n terms in blocks of at most 64 a thread and
then a tree by (64 + 20) u; so log Z by (D + 4 + 84) u absolute over terms that weigh, at
most 2^-17 for the spreads used here (terms with D > 30 weigh less than e^-30 n), and
x - M - log Z adds 2 u of its magnitude.  The entropy's sum weighs the same errors with
|d| e^d, at most D: 2^-17 (1 + H) + 2^-17."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def score(*a, **kw):
    from latentserve_amd.kernels import logprobs
    return logprobs.token_logprobs(*a, **kw)


def oracle(x, tok, top):
    """x [rows, n] numpy; (logprob, entropy, top values, top ids) in 64 bits."""
    with np.errstate(divide="ignore", invalid="ignore"):
        d = x.astype(np.float64)
        m = d.max(-1, keepdims=True)
        m = np.where(np.isneginf(m), 0, m)
        z = np.exp(d - m).sum(-1, keepdims=True)
        logp = np.where(np.isneginf(d), -np.inf, d - m - np.log(z))
        p = np.exp(logp)
        ent = -np.where(p > 0, p * logp, 0).sum(-1)
    r = np.arange(len(x))
    lp = np.where((tok >= 0) & (tok < x.shape[1]), logp[r, np.clip(tok, 0, x.shape[1] - 1)], 0)
    ids = np.argsort(-d, axis=-1, kind="stable")[:, :top]
    return lp, ent, np.take_along_axis(logp, ids, -1), ids


def close(got, want, tol):
    got = got.double().cpu().numpy()
    same = (got == want)                          # infinities
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got - want) <= tol(want))).all(), (got, want)


def check(x, tok, top):
    out = score(torch.from_numpy(x).cuda(), torch.from_numpy(tok).cuda(), top)
    lp, ent, tv, ti = oracle(x, tok, top)
    tol = lambda w: 2.0 ** -17 + 2.0 ** -23 * np.abs(w)  # noqa: E731
    close(out.logprob, lp, tol)
    close(out.entropy, ent, lambda w: 2.0 ** -16 + 2.0 ** -17 * w)
    if top:
        np.testing.assert_array_equal(out.top_ids.cpu().numpy(), ti)
        close(out.top_logprobs, tv, tol)
    else:
        assert out.top_logprobs is None and out.top_ids is None


def logits(rows, n, seed, dtype):
    g = np.random.default_rng(seed)
    x = 2.5 * g.standard_normal((rows, n))
    x[np.arange(rows), g.integers(0, n, rows)] += 8
    return x.astype(dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 2), (3, 7), (2, 255), (5, 1000), (1, 4097), (2, 16377),
                                    (2, 16384), (3, 16385), (1, 32003), (4, 151936), (1, 600001)])
def test_matches_64_bits(rows, n, dtype):
    g = np.random.default_rng(n)
    x, tok = logits(rows, n, n + rows, dtype), g.integers(0, n, rows)
    for top in sorted({0, 1, min(5, n), min(32, n)}):
        print(f"score rows={rows} n={n} top={top}", flush=True)
        check(x, tok, top)


def test_many_rows():
    check(logits(3001, 1003, 1, np.float16), np.random.default_rng(2).integers(0, 1003, 3001), 3)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [40, 5003, 50001])
def test_ties_go_to_the_lower_number(n, dtype):
    g = np.random.default_rng(n)
    x = np.stack((np.zeros(n), np.full(n, -3.0), g.integers(0, 3, n), np.arange(n) // 64 % 2,
                  -(np.arange(n) // 1000.0), np.arange(n) / 1000.0,
                  np.where(np.arange(n) % 2, 0.0, -0.0))).astype(dtype)
    check(x, np.zeros(len(x), np.int64) + 5, 32)


@pytest.mark.parametrize("n", [33, 20000, 70001])
def test_the_best_in_few_threads(n):
    """Runs of adjacent and of strided large entries: many candidates in one thread."""
    x = np.full((3, n), -10, np.float32)
    x[0, :33] = np.arange(33)
    x[1, ::max(1, 2048 * 8 // 64 // 8)] = 1
    x[2, n // 2:n // 2 + 16] = 3
    for dtype in (np.float16, np.float32):
        check(x.astype(dtype), np.array([0, 3, n // 2]), 32)


@pytest.mark.parametrize("n", [50, 40000])
def test_masked_logits(n):
    x = logits(5, n, 3, np.float32)
    x[0, 3:] = -np.inf                             # three left
    x[1] = -np.inf                                 # none
    x[2, ::2] = -np.inf
    x[3, 1:] = np.finfo(np.float32).min            # the type's lowest value
    x[4] = np.finfo(np.float32).min
    tok = np.array([1, 4, 2, 0, n - 1])
    check(x, tok, 5)
    h = x.copy()
    h[3, 1:] = h[4] = -65504
    check(h.astype(np.float16), tok, 5)


def test_padding_tokens_and_nan():
    n = 3000
    x = logits(6, n, 4, np.float16)
    x[2, 100] = np.nan
    x[3, 7] = np.inf
    tok = np.array([-1, n, 5, 6, -(1 << 40), 2])
    out = score(torch.from_numpy(x).cuda(), torch.from_numpy(tok).cuda(), 3)
    lp = out.logprob.cpu().numpy()
    assert lp[0] == lp[1] == lp[4] == 0
    assert np.isnan(lp[2]) and np.isnan(lp[3]) and np.isfinite(lp[5])
    assert out.top_ids[2, 0].item() == 100 and out.top_ids[3, 0].item() == 7
    assert np.isnan(out.entropy[2:4].cpu().numpy()).all()
    keep = [0, 1, 4, 5]
    want = oracle(x[keep], tok[keep], 3)
    close(out.entropy[keep], want[1], lambda w: 2.0 ** -16 + 2.0 ** -17 * w)
    np.testing.assert_array_equal(out.top_ids[keep].cpu().numpy(), want[3])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n,every", [(50, 7), (5003, 3), (40000, 1), (40000, 611), (151936, 9001)])
def test_nan_and_infinity_rank_first(n, every, dtype):
    """NaN, then +inf, then the rest, of each the lower numbers first."""
    x = logits(3, n, n, np.float32)
    x[0, ::every] = np.nan
    x[1, ::every] = np.inf
    x[1, n - 2] = np.nan
    x[2, ::every] = np.inf
    x[2, :n // 2] -= 40                            # negative ones
    x = x.astype(dtype)
    out = score(torch.from_numpy(x).cuda(), torch.zeros(3, dtype=torch.int64, device="cuda"), 32)
    rank = np.where(np.isnan(x), np.inf, np.where(np.isinf(x), 1e30, x.astype(np.float64)))
    want = np.argsort(-rank, axis=1, kind="stable")[:, :32]
    np.testing.assert_array_equal(out.top_ids.cpu().numpy(), want)
    for t in (out.logprob, out.entropy, out.top_logprobs):
        assert torch.isnan(t).all()


@pytest.mark.parametrize("n", [300, 151936])
def test_negative_halves(n):
    """Neighbouring negative fp16 values: where a bound of fewer bits takes in one more."""
    x = -(1 + np.random.default_rng(n).integers(0, 1024, (4, n)) / 1024).astype(np.float16)
    x[1] *= np.float16(2.0 ** -15)                 # subnormal ones
    x[2] = -x[2]
    x[3] *= np.float16(8192)
    check(x, np.array([0, 1, 2, n - 1]), 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strides_shapes_and_odd_starts(dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(4, 3, 20011, generator=g, device="cuda").to(dtype)
    for x in (wide[:, 1, 3:], wide[:, :, 1:1000], wide[1:, 0, :17], wide[..., ::2], wide[0, 0],
              wide.transpose(0, 1), wide[:0, 0]):
        tok = torch.randint(0, x.shape[-1], x.shape[:-1], generator=g, device="cuda")
        out = score(x, tok, 4)
        assert out.logprob.shape == out.entropy.shape == x.shape[:-1]
        assert out.top_ids.shape == out.top_logprobs.shape == x.shape[:-1] + (4,)
        if x.numel() == 0:
            continue
        flat = x.reshape(-1, x.shape[-1]).cpu().numpy()
        lp, ent, tv, ti = oracle(flat, tok.reshape(-1).cpu().numpy(), 4)
        np.testing.assert_array_equal(out.top_ids.reshape(-1, 4).cpu().numpy(), ti)
        close(out.logprob.reshape(-1), lp, lambda w: 2.0 ** -17 + 2.0 ** -23 * np.abs(w))


def test_streams_and_graphs_beside_each_other():
    xs = [logits(5, 60001, 10 + i, np.float16) for i in range(3)]
    toks = [np.arange(5) + i for i in range(3)]
    dx = [torch.from_numpy(x).cuda() for x in xs]
    dt = [torch.from_numpy(t).cuda() for t in toks]
    score(dx[0], dt[0], 5)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(score(dx[i], dt[i], 5))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for rep in range(4):
        for x in dx[:2]:
            x.neg_()
        for x in xs[:2]:
            np.negative(x, out=x)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = score(dx[2], dt[2], 5)
        torch.cuda.synchronize()
        for i, out in enumerate(outs + [eager]):
            lp, ent, tv, ti = oracle(xs[i], toks[i], 5)
            np.testing.assert_array_equal(out.top_ids.cpu().numpy(), ti)
            close(out.logprob, lp, lambda w: 2.0 ** -17 + 2.0 ** -23 * np.abs(w))
            close(out.entropy, ent, lambda w: 2.0 ** -16 + 2.0 ** -17 * w)
