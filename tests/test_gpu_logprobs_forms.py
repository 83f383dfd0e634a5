"""Every form of the log-probability kernel against 64 bits, on an MI355X: rows streamed
(no alternatives, more than 64 parts of 16384), rows held 64 logits a thread, in one part
and in several, and the short parts of small calls; fp16 and fp32, at odd starts, with
masks, ties, maxima that move, infinities and NaN.

Bounds, u = 2^-24 (half a step of fp32) and T the terms that a thread sums: an exponential
that weighs (of at most 2^-30, D = 44 units of log2) is off by (D + 4) u relative, its
thread's sum by T u, each of at most T / 32 moves to another maximum by 8 u, and the sums
over threads and parts by 30 u: log Z by A = (80 + 1.25 T) u.  x - M - log Z adds roundings
at its size, and the two factors between log2 and natural units theirs: 2^-22 of it.  The
entropy's sum has the same errors, each term weighed with |d| p, so A (1 + H) in the sum
and in log Z."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]

U = 2.0 ** -24
KINDS = 13


def score(*a, **kw):
    from latentserve_amd.kernels import logprobs
    return logprobs.token_logprobs(*a, **kw)


def form(rows, n, top):
    """(form, parts of a row, logits of a thread) by the rule; the parts checked against the
    library's workspace."""
    from latentserve_amd import _serving

    count = lambda size: -(-(n + 7) // size)  # noqa: E731
    if rows * count(16384) <= 64:
        got = "short", count(4096), 16
    elif top:
        got = "held", count(16384), 64
    else:
        size = -(-((n + 7) // -(-512 // rows)) // 16384) * 16384
        got = "streamed", count(size), min(size, n + 7) // 256 + 8
    need = _serving.lib().ls_token_logprobs_workspace_bytes(rows, n, top)
    assert need == (0 if got[1] == 1 else rows * got[1] * (4 + 2 * top) * 4)
    return got


def logits(rows, n, dtype, seed):
    """Row i of kind i % KINDS."""
    g = torch.Generator("cuda").manual_seed(seed)
    low, at = torch.finfo(dtype).min, torch.arange(n, device="cuda")
    x = (2.5 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    for i in range(rows):
        k, r = i % KINDS, x[i]
        if k == 1:
            r[:] = 0
        elif k == 2:
            r[:] = -3
        elif k == 3:
            r[:] = torch.randint(0, 3, (n,), generator=g, device="cuda")
        elif k == 4:
            r[:] = -np.inf
        elif k == 5:
            r[:] = -np.inf
            r[[0, n // 2, n - 1]] = torch.tensor([1.0, -2.0, 0.5], dtype=dtype, device="cuda")
        elif k == 6:
            r[:] = low
            r[(7 * i) % n] = 3
        elif k == 7:
            r[:] = low
        elif k == 8:
            r[:] = -(at / max(n, 2) * 40)
        elif k == 9:
            r[:] = at / max(n, 2) * 40               # the maximum moves to the end
        elif k == 10:
            r[::2] = -np.inf
        elif k == 11:
            r[:] = at // 64 % 2
        elif k == 12:
            r *= 20000 / 2.5 if dtype == torch.float16 else 1e7
            r.clamp_(-60000, 60000) if dtype == torch.float16 else None
    return x


def oracle(x, tok, top):
    d = x.double()
    m = d.amax(-1, keepdim=True)
    m = torch.where(m == -np.inf, torch.zeros_like(m), m)
    e = torch.exp(d - m)
    z = e.sum(-1, keepdim=True)
    lz = torch.log(z)
    logp = torch.where(d == -np.inf, d, d - m - lz)
    ent = -torch.where(e > 0, e / z * logp, torch.zeros_like(e)).sum(-1)
    ent = torch.where(z[:, 0] == 0, torch.zeros_like(ent), ent)
    ids = torch.sort(d, dim=-1, descending=True, stable=True)[1][:, :top]
    inside = (tok >= 0) & (tok < x.shape[1])
    lp = logp.gather(1, tok.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    return torch.where(inside, lp, torch.zeros_like(lp)), ent, logp.gather(1, ids), ids


def near(got, want, tol, what):
    same = got.double() == want                       # infinities
    bad = ~(same | ((got.double() - want).abs() <= tol))
    assert not bad.any(), (what, bad.nonzero()[:4].tolist(), got[bad][:4].tolist(),
                           want[bad][:4].tolist())


def check(x, tok, top, terms):
    out = score(x, tok, top)
    lp, ent, tv, ti = oracle(x, tok, top)
    a = (80 + 1.25 * terms) * U
    near(out.logprob, lp, a + 2.0 ** -22 * lp.abs(), "logprob")
    near(out.entropy, ent, 2 * a * (1 + ent), "entropy")
    if top:
        assert torch.equal(out.top_ids, ti)
        near(out.top_logprobs, tv, a + 2.0 ** -22 * tv.abs(), "top")
    again = score(x, tok, top)
    for p, q in zip(out, again):
        assert p is None or torch.equal(p, q)         # (repeats bit for bit)
    return out


def tokens(rows, n, seed):
    tok = torch.randint(0, n, (rows,), generator=torch.Generator().manual_seed(seed))
    tok[::7], tok[3::11], tok[5::13] = 0, n - 1, -1
    return tok.cuda()


CASES = [("streamed", 65, 1, 0), ("streamed", 70, 7, 0), ("streamed", 70, 1003, 0),
         ("streamed", 67, 16377, 0), ("streamed", 67, 16385, 0), ("streamed", 13, 151936, 0),
         ("streamed", 2, 600001, 0), ("streamed", 300, 50001, 0), ("streamed", 200, 151936, 0),
         ("streamed", 600, 40001, 0), ("streamed", 1300, 8191, 0), ("streamed", 65, 8200, 0),
         ("held", 66, 40, 32), ("held", 70, 1003, 5), ("held", 65, 16377, 32),
         ("held", 65, 16378, 1), ("held", 16, 151936, 20), ("held", 30, 50001, 32),
         ("held", 30, 50001, 1), ("held", 2, 600001, 32), ("held", 2, 1200001, 32),
         ("short", 3, 16384, 0), ("short", 13, 40001, 32), ("short", 1, 600001, 5)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("want,rows,n,top", CASES, ids=lambda v: str(v))
def test_a_form(want, rows, n, top, dtype):
    got, parts, terms = form(rows, n, top)
    assert got == want
    print(f"{want} rows={rows} n={n} top={top} parts={parts}", flush=True)
    check(logits(rows, n, dtype, n), tokens(rows, n, n), top, terms)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("rows,n,top", [(70, 1003, 0), (67, 16400, 0), (171, 66000, 0),
                                        (70, 1003, 5), (40, 33000, 32)])
@pytest.mark.parametrize("first,gap", [(1, 0), (3, 2), (7, 9)])
def test_rows_at_odd_starts(rows, n, top, first, gap, dtype):
    """Rows that start at any element, the next one's start another."""
    wide = logits(rows, n + first + gap, dtype, 3)
    wide[:, :first], wide[:, first + n:] = np.inf, np.nan          # nobody reads these
    x = wide[:, first:first + n]
    assert form(rows, n, top)[0] == ("held" if top else "streamed")
    print(f"odd rows={rows} n={n} top={top} start={first}", flush=True)
    check(x, tokens(rows, n, 1), top, form(rows, n, top)[2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("rows,n,top", [(70, 1003, 0), (68, 16385, 0), (20, 151936, 0),
                                        (70, 1003, 32), (20, 60001, 32), (66, 16384, 5)])
def test_nan_and_infinity(rows, n, top, dtype):
    """A NaN or +inf makes its row NaN wherever it lies and leaves the others; it ranks
    first, NaN before +inf."""
    x, tok = logits(rows, n, dtype, 9), tokens(rows, n, 2)
    places = [0, n - 1, n // 2, min(16383, n - 1), min(16384, n - 1), 255, 8 * 256 % n]
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i in range(1, rows, 2):
        bad[i] = True
        at = places[i // 2 % len(places)]
        if i % 4 == 1:
            x[i, at] = np.nan
        else:
            x[i, at] = np.inf
        if i % 5 == 0:                                 # many of both
            x[i, ::3], x[i, 1::7] = np.inf, np.nan
    print(f"nan rows={rows} n={n} top={top} {form(rows, n, top)}", flush=True)
    out = score(x, tok, top)
    lp = torch.where((tok >= 0) & (tok < n), out.logprob, torch.full_like(out.logprob, np.nan))
    assert torch.isnan(lp[bad]).all() and torch.isnan(out.entropy[bad]).all()
    assert (out.logprob[tok < 0] == 0).all()
    if top:
        assert torch.isnan(out.top_logprobs[bad]).all()
        # (NaN as the largest of 64 bits, +inf below it)
        d = torch.where(torch.isnan(x), torch.full_like(x, 2, dtype=torch.float64) * 1e300,
                        torch.where(x == np.inf, torch.full_like(x, 1, dtype=torch.float64) * 1e300,
                                    x.double()))
        ids = torch.sort(d, dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(out.top_ids, ids)
    keep = ~bad
    want = oracle(x[keep], tok[keep], top)
    a = (80 + 1.25 * form(rows, n, top)[2]) * U
    near(out.logprob[keep], want[0], a + 2.0 ** -22 * want[0].abs(), "logprob")
    near(out.entropy[keep], want[1], 2 * a * (1 + want[1]), "entropy")


@pytest.mark.parametrize("rows,n,top", [(13, 151936, 0), (200, 70001, 0), (20, 60001, 20)])
def test_captured_calls_replay(rows, n, top):
    """Parts of a row handed over in a graph, its inputs changed between replays, beside
    eager calls of other sizes."""
    x, tok = logits(rows, n, torch.float16, 4), tokens(rows, n, 4)
    score(x, tok, top)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [score(x, tok, top) for _ in range(2)]
    for rep in range(4):
        x.copy_(logits(rows, n, torch.float16, 5 + rep))
        eager = score(x, tok, top)
        torch.cuda.synchronize()
        g.replay()
        score(x[:2], tok[:2], 3)
        torch.cuda.synchronize()
        for out in outs:
            for p, q in zip(out, eager):
                assert p is None or torch.equal(p, q), rep
