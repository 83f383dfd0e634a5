"""Weight sums, accepted paths, selection and moves against numpy in 64 bits
(tests/tree_ref.py), on an MI355X."""

from __future__ import annotations

import numpy as np
import pytest

from tests import tree_ref as ref
from tests.test_gpu_tree_attention import case, dev

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def ce():
    from latentserve_amd.kernels.hip import cache_eviction
    return cache_eviction


def ta():
    from latentserve_amd.kernels.hip import tree_attention
    return tree_attention


def some_sums(rows, h, length, seed):
    return np.random.default_rng(seed).random((rows, h, length)).astype(np.float32)


# ---- decode attention that adds its weights ----------------------------------------


@pytest.mark.parametrize("lens,h,r", [([1], 1, 1), ([16, 0, 17], 2, 6), ([2048], 2, 6), ([700, 33, 255, 1], 3, 16),
                                      ([5000], 1, 7), ([256, 257, 64], 2, 2), ([20011], 1, 4)])
def test_decode_weights(lens, h, r):
    q, k, v, t, l, _ = case(lens, 1, h, r, 30 + r)
    width = t.shape[1] * 16
    sums = some_sums(len(lens) + 2, h, width, 1)
    rows = np.random.default_rng(2).permutation(len(lens) + 2)[:len(lens)].astype(np.int32)
    sd = dev(sums)
    print(f"decode weights {lens} h={h} r={r}", flush=True)
    out = ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), sd, dev(rows))
    want, lse, tol, _ = ref.attend(q, k, v, t, l)
    assert (np.abs(out.double().cpu().numpy() - want[:, 0]) <= tol[:, 0]).all()
    path = np.zeros((len(lens), 1), np.int32)
    add, atol = ref.path_weights(q, lse, k, t, l, path, np.ones(len(lens), np.int32))
    exp, bound = sums.astype(np.float64), np.zeros_like(sums, np.float64)
    n = add.shape[2]
    exp[rows, :, :n] += add
    # (the row's own statistic was made in 32 bits too: its bound, relative)
    bound[rows, :, :n] = 2 * atol + add * 2.0 ** -16 + 2 * ref.SINGLE * exp[rows, :, :n]
    got = sd.double().cpu().numpy()
    assert (np.abs(got - exp) <= bound).all(), np.abs(got - exp).max()
    for i, length in enumerate(lens):
        if length:                                           # a row of weights is one
            total = (got[rows[i], :, :length] - sums[rows[i], :, :length]).sum(-1)
            np.testing.assert_allclose(total, r, rtol=1e-4)


def test_decode_weights_of_no_rows_and_short_sums():
    q, k, v, t, l, _ = case([200, 100, 40], 1, 2, 6, 31)
    full = dev(some_sums(3, 2, 208, 3))
    short = full[:, :, :90].clone()
    rows = dev(np.array([2, -1, 7], np.int32))
    before = full.clone()
    a = ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), full, rows)
    assert torch.equal(full[:2], before[:2]) and not torch.equal(full[2], before[2])
    b = ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), short, rows)
    assert torch.equal(a, b) and torch.equal(short[2], full[2, :, :90])


def test_decode_weights_equals_the_decode():
    """Beside the framework's own decode, on the same cache: one rounding of fp16 apart."""
    from latentserve_amd.kernels.gqa.paged_decode import paged_decode_attention
    q, k, v, t, l, _ = case([1000, 2048, 37], 1, 2, 6, 32)
    a = ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l),
                                  torch.zeros(3, 2, 2048, device="cuda"))
    b = paged_decode_attention(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), max_seq_len=2048)
    assert float((a.float() - b.float()).abs().max()) < 2e-3


# ---- accepted paths' weights ----------------------------------------------------------


@pytest.mark.parametrize("lens,n,h,r,most", [([9], 4, 1, 1, 1), ([300, 20, 0, 5], 8, 2, 6, 5), ([33, 64, 4], 16, 3, 4, 12),
                                             ([4000], 16, 2, 6, 5), ([600, 70], 70, 1, 16, 64), ([31, 32, 300], 3, 2, 8, 3)])
def test_add_weights(lens, n, h, r, most):
    rng = np.random.default_rng(33)
    q, k, v, t, l, _ = case(lens, n, h, r, 34)
    b = len(lens)
    path = np.stack([np.sort(rng.permutation(n)[:most]) for _ in range(b)]).astype(np.int32)
    lengths = rng.integers(0, most + 1, b).astype(np.int32)
    lengths[0] = most
    lse = (rng.standard_normal((b, n, h, r)) + 8).astype(np.float32)
    if most > 1:
        path[0, 0], lse[0, path[0, 1], 0, 0] = n + 3, -np.inf   # no node; a row that saw nothing
    sums = some_sums(b + 1, h, t.shape[1] * 16, 4)
    rows = rng.permutation(b + 1)[:b].astype(np.int32)
    sd = dev(sums)
    print(f"add weights {lens} n={n} most={most}", flush=True)
    ce().add_weights(dev(q), dev(lse), dev(k), dev(t), dev(l), sd, dev(rows), dev(path), dev(lengths))
    add, tol = ref.path_weights(q, lse, k, t, l, path, lengths)
    exp, bound = sums.astype(np.float64), np.zeros_like(sums, np.float64)
    exp[rows, :, :add.shape[2]] += add
    bound[rows, :, :add.shape[2]] = tol + ref.SINGLE * 2 * exp[rows, :, :add.shape[2]]
    got = sd.double().cpu().numpy()
    over = np.abs(got - exp) - bound
    assert (over <= 0).all(), over.max()


def test_add_weights_without_a_path_is_a_chain():
    q, k, v, t, l, _ = case([100, 7], 6, 2, 4, 35)
    lse = torch.empty(2, 6, 2, 4, device="cuda")
    ta().tree_attention(dev(q), dev(k), dev(v), dev(t), dev(l), lse=lse)
    a, b = torch.zeros(2, 2, 112, device="cuda"), torch.zeros(2, 2, 112, device="cuda")
    ce().add_weights(dev(q), lse, dev(k), dev(t), dev(l), a)
    path = dev(np.tile(np.arange(6, dtype=np.int32), (2, 1)))
    ce().add_weights(dev(q), lse, dev(k), dev(t), dev(l), b, path=path)
    assert torch.equal(a, b)
    np.testing.assert_allclose(a.sum(-1).cpu().numpy(), 6 * 4, rtol=1e-4)


def test_add_weights_passes_by_blocks_outside_the_pool_and_infinities():
    q, k, v, t, l, _ = case([300, 80], 4, 2, 6, 36)
    lse = np.full((2, 4, 2, 6), 9, np.float32)
    t[0, 3], t[1, 0] = -1, k.shape[0]
    lengths = np.array([2, 3], np.int32)
    path = np.array([[0, 3], [0, 1]], np.int32)
    lengths[1] = 2
    sd = torch.zeros(2, 2, t.shape[1] * 16, device="cuda")
    ce().add_weights(dev(q), dev(lse), dev(k), dev(t), dev(l), sd, path=dev(path), lengths=dev(lengths))
    add, tol = ref.path_weights(q, lse, k, t, l, path, lengths)
    got = sd.double().cpu().numpy()[:, :, :300]
    assert (np.abs(got - add) <= tol + 2 * ref.SINGLE * add).all()
    # a key of minus infinity to every row that is there gets nothing, not a NaN from the
    # padding rows
    k2 = k.copy()
    q2 = np.abs(q)
    blk = t[0, 5]
    k2[blk, 7] = -np.inf
    sd.zero_()
    ce().add_weights(dev(q2), dev(lse), dev(k2), dev(t), dev(l), sd, path=dev(path), lengths=dev(lengths))
    assert torch.isfinite(sd).all() and (sd[0, :, 87] == 0).all()


# ---- acceptance -------------------------------------------------------------------------


def drafted(b, n, seed, agree=0.8, values=3):
    rng = np.random.default_rng(seed)
    parents = np.stack([ref.random_tree(n, rng) for _ in range(b)])
    tokens = rng.integers(0, values, (b, n)).astype(np.int64)
    choices = rng.integers(0, values, (b, n)).astype(np.int64)
    for i in range(b):
        for j in range(1, n):
            if rng.random() < agree:
                choices[i, parents[i, j]] = tokens[i, j]
    return tokens, parents, choices


@pytest.mark.parametrize("b,n,h,layers", [(1, 1, 1, 1), (3, 7, 2, 2), (5, 64, 1, 3), (2, 65, 3, 1), (4, 130, 2, 33),
                                          (2, 256, 1, 2)])
def test_accept_tokens(b, n, h, layers):
    rng = np.random.default_rng(40 + n)
    tokens, parents, choices = drafted(b, n, 41 + n)
    counts = rng.integers(0, n + 1, b).astype(np.int32)
    counts[0] = n
    lens = np.array([n + int(x) for x in rng.integers(0, 60, b)], np.int32)
    width = int(-(-lens.max() // 16))
    nb = b * width + 2
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    pools = rng.integers(-2000, 2000, (2, layers, nb, 16, h, 128)).astype(np.float16)
    for use in (None, counts):
        dp = dev(pools)
        print(f"accept b={b} n={n} layers={layers} counts={use is not None}", flush=True)
        got = ta().accept_tokens(dev(tokens), dev(parents), dev(choices), list(dp[0]), list(dp[1]),
                                 dev(tables), dev(lens), None if use is None else dev(use))
        want = pools.copy()
        for i in range(b):
            path, nxt = ref.accepted(tokens[i], parents[i], choices[i], n if use is None else int(use[i]))
            assert got.path[i].tolist() == path + [-1] * (n - len(path))
            assert int(got.lengths[i]) == len(path) and int(got.next_tokens[i]) == nxt
            for j, node in enumerate(path):
                a, z = lens[i] - n + node, lens[i] - n + j
                want[:, :, tables[i, z // 16], z % 16] = pools[:, :, tables[i, a // 16], a % 16]
        np.testing.assert_array_equal(dp.cpu().numpy(), want)


def test_accept_of_a_whole_chain_moves_nothing():
    n = 40
    parents = np.arange(-1, n - 1, dtype=np.int32)[None]
    tokens = np.arange(n, dtype=np.int64)[None]
    choices = tokens + 1
    pools = torch.randn(2, 5, 16, 1, 128, device="cuda").half()
    before = pools.clone()
    table = torch.tensor([[3, 1, 4, 0]], dtype=torch.int32, device="cuda")
    got = ta().accept_tokens(dev(tokens), dev(parents), dev(choices), [pools[0]], [pools[1]], table,
                             torch.tensor([n + 9], dtype=torch.int32, device="cuda"))
    assert int(got.lengths[0]) == n and int(got.next_tokens[0]) == n
    assert torch.equal(pools, before)


# ---- selection and moves -----------------------------------------------------------------


def rank_sums(kind, shape, rng):
    w = rng.random(shape).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    if kind == "few values":
        return (rng.integers(0, 4, shape) / 4).astype(np.float32)
    if kind == "zeros of both signs":
        return np.where(rng.random(shape) < 0.5, np.float32(-0.0), np.float32(0.0)).astype(np.float32)
    if kind == "all numbers":
        w = (rng.standard_normal(shape) * 10.0 ** rng.integers(-40, 38, shape)).astype(np.float32)
        w[rng.random(shape) < 0.05] = np.inf
        w[rng.random(shape) < 0.05] = -np.inf
        w[rng.random(shape) < 0.03] = np.nan
    if kind == "close":
        w = (1 + rng.integers(0, 300, shape) * 2.0 ** -23).astype(np.float32)
    return w


@pytest.mark.parametrize("kind", ["random", "equal", "few values", "zeros of both signs", "all numbers", "close"])
@pytest.mark.parametrize("lens,budget,sinks,recent", [([1, 0, 5], 4, 1, 1), ([100, 64, 63, 65], 64, 4, 16),
                                                      ([1025, 1024, 30], 1000, 0, 0), ([5000, 2048], 700, 4, 175),
                                                      ([20011, 16385], 16384, 4, 4000), ([300], 1, 0, 0), ([300], 1, 1, 0),
                                                      ([777], 776, 0, 776), ([40000], 33, 3, 30)])
def test_select_tokens(kind, lens, budget, sinks, recent):
    rng = np.random.default_rng(50)
    b, h, layers = len(lens), 2, 2
    sums = rank_sums(kind, (layers, b, h, max(lens) + 5), rng)
    print(f"select {kind} {lens} {budget}", flush=True)
    keep, kept = ce().select_tokens(dev(sums), dev(np.array(lens, np.int32)), budget, sinks, recent)
    keep, kept = keep.cpu().numpy(), kept.cpu().numpy()
    for x in range(layers):
        for i in range(b):
            for y in range(h):
                want = ref.selected(sums[x, i, y], lens[i], budget, sinks, recent)
                m = len(want)
                assert keep[x, i, y, :m].tolist() == want and (keep[x, i, y, m:] == -1).all()
                np.testing.assert_array_equal(kept[x, i, y, :m], sums[x, i, y][want])
                assert (kept[x, i, y, m:] == 0).all()


def test_select_takes_strided_sums_and_lengths_past_them():
    rng = np.random.default_rng(51)
    wide = dev(rng.random((2, 5, 3, 200)).astype(np.float32))
    view = wide[:, 1:4, ::2, 10:110]
    lens = dev(np.array([90, 100, 5000], np.int32))
    a = ce().select_tokens(view, lens, 50, 2, 10)
    b = ce().select_tokens(view.contiguous(), lens.clamp(max=100), 50, 2, 10)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("lens,budget,h,layers", [([50, 16, 1, 0], 17, 2, 2), ([1000, 700], 400, 1, 3), ([300], 1, 3, 1),
                                                  ([3000, 2999, 12], 2500, 2, 1), ([40, 70], 33, 1, 40)])
def test_evict_moves_what_it_keeps(lens, budget, h, layers):
    rng = np.random.default_rng(52)
    b = len(lens)
    width = -(-max(lens) // 16) + 1
    nb = b * width + 2
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    pools = rng.integers(-2000, 2000, (2, layers, nb, 16, h, 128)).astype(np.float16)
    sums = rng.random((layers, b, h, width * 16)).astype(np.float32)
    dp = dev(pools)
    print(f"evict {lens} {budget} layers={layers}", flush=True)
    keep, kept = ce().evict_tokens(dev(sums), list(dp[0]), list(dp[1]), dev(tables),
                                   dev(np.array(lens, np.int32)), budget, sinks=min(2, budget), recent=budget // 3)
    want = pools.copy()
    for x in range(layers):
        for i in range(b):
            for y in range(h):
                pos = ref.selected(sums[x, i, y], lens[i], budget, min(2, budget), budget // 3)
                assert keep[x, i, y, :len(pos)].tolist() == pos
                src = np.array(pos, int)
                dst = np.arange(len(pos))
                want[:, x, tables[i, dst // 16], dst % 16, y] = pools[:, x, tables[i, src // 16], src % 16, y]
    np.testing.assert_array_equal(dp.cpu().numpy(), want)


def test_evict_passes_by_blocks_outside_the_pool():
    rng = np.random.default_rng(53)
    pools = rng.integers(-2000, 2000, (2, 6, 16, 1, 128)).astype(np.float16)
    tables = np.array([[0, 9, 2, -1, 4]], np.int32)
    dp = dev(pools)
    sums = np.zeros((1, 1, 1, 80), np.float32)
    sums[..., [16, 20, 35, 50, 70]] = 5
    keep, _ = ce().evict_tokens(dev(sums), [dp[0]], [dp[1]], dev(tables), dev(np.array([80], np.int32)), 5, 0, 0)
    assert keep[0, 0, 0].tolist() == [16, 20, 35, 50, 70]
    want = pools.copy()
    want[:, 0, 2], want[:, 0, 4] = pools[:, 2, 3], pools[:, 4, 6]        # 35 and 70: the others have no page
    np.testing.assert_array_equal(dp.cpu().numpy(), want)


# ---- together, as a serving step uses them ---------------------------------------------------


def test_a_tree_step_and_an_eviction_together():
    """Drafts checked, the path kept, its weights added, a decode step, then eviction: the
    cache and the sums against the definitions, and against a cache that never held the
    rejected nodes."""
    rng = np.random.default_rng(60)
    b, n, h, r, layers = 3, 9, 2, 4, 2
    ctx = [70, 33, 128]
    lens = np.array([c + n for c in ctx], np.int32)
    width = 16
    nb = b * width + 1
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    pools = rng.standard_normal((2, layers, nb, 16, h, 128)).astype(np.float16)
    tokens, parents, choices = drafted(b, n, 61)
    q = rng.standard_normal((layers, b, n, h, r, 128)).astype(np.float16)
    dp, dt, dl = dev(pools), dev(tables), dev(lens)
    masks, _ = ta().tree_masks(dev(parents))
    lse = torch.empty(layers, b, n, h, r, device="cuda")
    seen = np.stack([ref.seen_by(p) for p in parents])
    outs = []
    for x in range(layers):
        outs.append(ta().tree_attention(dev(q[x]), dp[0, x], dp[1, x], dt, dl, masks, lse=lse[x]))
        want, _, tol, _ = ref.attend(q[x], pools[0, x], pools[1, x], tables, lens, seen)
        assert (np.abs(outs[x].double().cpu().numpy() - want) <= tol).all()
    got = ta().accept_tokens(dev(tokens), dev(parents), dev(choices), list(dp[0]), list(dp[1]), dt, dl)
    lengths = got.lengths.cpu().numpy()
    after = np.array(ctx, np.int32) + lengths
    da = dev(after)
    # a chain of the path's queries over the cache as it is now gives the tree's rows
    for x in range(layers):
        for i in range(b):
            p = got.path[i, :lengths[i]].long()
            qi = dev(q[x])[i, p][None].contiguous()
            again = ta().tree_attention(qi, dp[0, x], dp[1, x], dt[i:i + 1].contiguous(), da[i:i + 1].contiguous())
            diff = (again[0].float() - outs[x][i, p].float()).abs().max()
            assert float(diff) <= 2 * 2.0 ** -10 * float(outs[x][i, p].float().abs().max())
    sums = torch.zeros(layers, b, h, width * 16, device="cuda")
    for x in range(layers):
        ce().add_weights(dev(q[x]), lse[x], dp[0, x], dt, da, sums[x], path=got.path, lengths=got.lengths)
    np.testing.assert_allclose(sums.sum(-1).cpu().numpy(), np.broadcast_to(lengths[None, :, None] * r, (layers, b, h)),
                               rtol=1e-4)
    q1 = dev(rng.standard_normal((b, h, r, 128)).astype(np.float16))
    for x in range(layers):
        ce().paged_decode_weights(q1, dp[0, x], dp[1, x], dt, da, sums[x])
    budget = 40
    state, now = sums.cpu().numpy(), dp.cpu().numpy()
    keep, kept = ce().evict_tokens(sums, list(dp[0]), list(dp[1]), dt, da, budget)
    for x in range(layers):
        for i in range(b):
            for y in range(h):
                pos = ref.selected(state[x, i, y], after[i], budget, 4, 10)
                assert keep[x, i, y, :len(pos)].tolist() == pos
    # attention over what is left is attention over those rows alone
    left = np.minimum(after, budget).astype(np.int32)
    o = ta().tree_attention(q1[:, None], dp[0, 0], dp[1, 0], dt, dev(left))
    kk, vv = now[0, 0], now[1, 0]
    for i in range(b):
        for y in range(h):
            pos = np.array(keep[0, i, y, :left[i]].tolist())
            ks, vs = kk[tables[i, pos // 16], pos % 16, y], vv[tables[i, pos // 16], pos % 16, y]
            qq = q1[i, y].double().cpu().numpy()
            s = qq @ ks.astype(np.float64).T * 128 ** -0.5
            p = np.exp(s - s.max(-1, keepdims=True))
            want = p @ vs.astype(np.float64) / p.sum(-1, keepdims=True)
            assert np.abs(o[i, 0, y].double().cpu().numpy() - want).max() < 2e-3


@pytest.mark.parametrize("n", [2, 12, 40])
def test_captured_and_replayed_with_eager_work_between(n):
    """Two graphs and eager calls in turn, each replay against the eager result."""
    q, k, v, t, l, seen = case([400, 90, n], n, 2, 6, 70)
    dq, dk, dv, dt, dl = (dev(x) for x in (q, k, v, t, l))
    words = dev(ref.words_of(seen))
    want = ta().tree_attention(dq, dk, dv, dt, dl, words)
    q1 = dq[:, 0].contiguous()
    base = torch.zeros(3, 2, t.shape[1] * 16, device="cuda")
    want1 = ce().paged_decode_weights(q1, dk, dv, dt, dl, base)
    sums = torch.zeros_like(base)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = ta().tree_attention(dq, dk, dv, dt, dl, words)
            sums.zero_()
            o1 = ce().paged_decode_weights(q1, dk, dv, dt, dl, sums)
        graphs.append(g)
        outs.append((o, o1))
    for turn in range(4):
        for g, (o, o1) in zip(graphs, outs):
            o.zero_()
            sums.fill_(5)
            print(f"replay {turn}", flush=True)
            g.replay()
            eager = ta().tree_attention(dq, dk, dv, dt, dl, words)
            torch.cuda.synchronize()
            assert torch.equal(o, want) and torch.equal(eager, want)
            assert torch.equal(o1, want1) and torch.equal(sums, base)


def test_two_streams_at_once():
    cases = [[dev(x) for x in case([3000, 500], 16, 2, 6, 80 + i)] for i in range(2)]
    words = [dev(ref.words_of(c[5].cpu().numpy())) for c in cases]
    want = [ta().tree_attention(*c[:5], w) for c, w in zip(cases, words)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for c, w, s in zip(cases, words, streams):
            with torch.cuda.stream(s):
                got.append(ta().tree_attention(*c[:5], w))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
