"""Attention of drafted trees against numpy in 64 bits (tests/tree_ref.py), on an
MI355X: shapes on both sides of every launch form, lengths of zero, one and odd ones,
masks that leave a row nothing, infinities and NaN where a row does not look."""

from __future__ import annotations

import numpy as np
import pytest

from tests import tree_ref as ref

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def ta():
    from latentserve_amd.kernels.hip import tree_attention
    return tree_attention


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def case(lens, n, h, r, seed, width=None):
    rng = np.random.default_rng(seed)
    b = len(lens)
    width = max(1, -(-max(lens) // 16)) if width is None else width
    nb = b * width + 3
    k = rng.standard_normal((nb, 16, h, 128)).astype(np.float16)
    v = rng.standard_normal((nb, 16, h, 128)).astype(np.float16)
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    q = (rng.standard_normal((b, n, h, r, 128)) * 2).astype(np.float16)
    seen = np.stack([ref.seen_by(ref.random_tree(n, rng)) for _ in range(b)])
    return q, k, v, tables, np.array(lens, np.int32), seen


def check(q, k, v, tables, lens, seen=None, counts=None, **kw):
    print(f"tree {q.shape} lens {lens.tolist()[:8]} {sorted(kw)}", flush=True)
    lse = torch.full(q.shape[:4], 7.0, device="cuda")
    out = ta().tree_attention(dev(q), dev(k), dev(v), dev(tables), dev(lens),
                              None if seen is None else dev(ref.words_of(seen)),
                              None if counts is None else dev(counts), lse=lse, **kw)
    torch.cuda.synchronize()
    want, wl, tol, ltol = ref.attend(q, k, v, tables, lens, seen, counts,
                                     kw.get("softmax_scale", 128.0 ** -0.5))
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    none = np.isneginf(wl)
    np.testing.assert_array_equal(np.isneginf(gl), none)
    assert (got[none] == 0).all()
    over = np.abs(got - want) - tol
    assert (over <= 0).all(), f"worst {over.max():.3g} past the bound at {np.argwhere(over > 0)[:4]}"
    lover = np.abs(gl - wl)[~none] - ltol[~none]
    assert (lover <= 0).all(), f"lse {lover.max():.3g} past the bound"
    return out, lse


# rows a head below, at and above 32, 64, 128 and 256; every n_rep
@pytest.mark.parametrize("n,r", [(1, 1), (1, 6), (5, 6), (8, 4), (33, 1), (9, 6), (16, 4), (13, 5),
                                 (16, 8), (43, 3), (32, 8), (37, 7), (70, 2), (65, 6), (128, 2),
                                 (129, 4), (256, 1)])
@pytest.mark.parametrize("h", [1, 2])
def test_tree_of_every_launch_form(n, r, h):
    lens = [n + 700, n, n + 1, n + 263]
    check(*case(lens, n, h, r, 10 * n + r))


@pytest.mark.parametrize("lens", [[1], [16], [17], [31, 32, 33], [128, 129, 127, 0], [0, 0], [255, 256, 257, 1]])
@pytest.mark.parametrize("n,r", [(1, 6), (3, 16), (12, 6), (40, 8)])
def test_lengths_from_zero(lens, n, r):
    """Lengths of zero, and ones below the number of nodes: no context, so many nodes."""
    check(*case(lens, n, 2, r, 3))


@pytest.mark.parametrize("n,r,h", [(6, 6, 2), (24, 6, 3), (64, 4, 1)])
def test_no_masks_is_a_chain(n, r, h):
    q, k, v, t, l, _ = case([n + 200, n, n + 3], n, h, r, 4)
    check(q, k, v, t, l)


@pytest.mark.parametrize("n,r", [(7, 4), (20, 6), (64, 6)])
def test_counts_leave_the_other_nodes_out(n, r):
    q, k, v, t, l, seen = case([300, 300, 77 + n, n, 140 + n], n, 2, r, 5)
    counts = np.array([n, 1, 0, n // 2, n + 5], np.int32)
    counts[3] = -2
    check(q, k, v, t, l, seen, counts)
    check(q, k, v, t, l, None, counts)


@pytest.mark.parametrize("n,r", [(5, 6), (16, 6), (30, 8)])
def test_rows_that_see_nothing(n, r):
    """Masks of no bits: a row sees its context alone, or, without one, nothing."""
    q, k, v, t, l, seen = case([n, n + 40, n], n, 2, r, 6)
    seen[0, ::2] = False
    seen[1, 1::3] = False
    seen[2] = False
    check(q, k, v, t, l, seen)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n,r", [(4, 6), (12, 5), (40, 4), (48, 8)])
def test_what_a_row_does_not_see_changes_nothing(n, r, bad):
    """Nodes that some rows see and others do not, rows past the end and other sequences'
    pages hold infinities or NaN: rows that do not see them are bit for bit as without."""
    lens = [n + 150, n + 16, n]
    q, k, v, t, l, seen = case(lens, n, 2, r, 7)
    clean, clse = check(q, k, v, t, l, seen)
    k2, v2 = k.copy(), v.copy()
    used = np.zeros(k.shape[:2], bool)
    for b, length in enumerate(lens):
        pos = np.arange(length)
        used[t[b, pos // 16], pos % 16] = True
    k2[~used], v2[~used] = bad, bad
    hidden = n // 2                                     # of sequence 0: its row and who sees it
    at = lens[0] - n + hidden
    k2[t[0, at // 16], at % 16, :, ::5] = bad
    v2[t[0, at // 16], at % 16, :, 3::7] = bad
    print(f"hidden n={n} r={r} {bad}", flush=True)
    lse = torch.empty_like(clse)
    out = ta().tree_attention(dev(q), dev(k2), dev(v2), dev(t), dev(l), dev(ref.words_of(seen)),
                              lse=lse)
    blind = ~seen[:, :, hidden]
    blind[1:] = True
    mask = torch.from_numpy(blind).cuda()
    # (products of a row at a time: the same sums, in their own order)
    assert torch.equal(lse[mask], clse[mask])
    want, _, tol, _ = ref.attend(q, k, v, t, l, seen)
    over = np.abs(out.double().cpu().numpy() - want) - tol
    assert (over[blind] <= 0).all()
    assert not torch.isfinite(out[0][~mask[0]].float()).all(-1).any()


def test_blocks_outside_the_pool_are_skipped():
    for n, r in ((3, 6), (10, 6), (20, 6), (40, 7)):
        q, k, v, t, l, seen = case([500, 333 + n, 64 + n], n, 2, r, 8)
        t[0, 3], t[0, 17], t[1, 0], t[2, 1] = -1, k.shape[0], 1 << 30, -7
        check(q, k, v, t, l, seen)


def test_tokens_past_the_table_are_not_there():
    q, k, v, t, l, seen = case([200, 100], 5, 2, 6, 9)
    check(q, k, v, t[:, :6].copy(), l, seen)


@pytest.mark.parametrize("n,r", [(2, 6), (16, 6), (64, 6)])
def test_long_axis_split_and_joined(n, r):
    check(*case([20011], n, 1, r, 11))


@pytest.mark.parametrize("n,r", [(4, 6), (33, 4)])
def test_many_sequences_of_all_lengths(n, r):
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 900, 70)]
    check(*case(lens, n, 2, r, 12))


def test_expected_length_only_sizes_the_launch():
    a = case([3000, 17, 2048], 9, 2, 6, 13)
    for m in (1, 100, 2048, 3000, 10 ** 9):
        check(*a, max_seq_len=m)


@pytest.mark.parametrize("scale", [1e-6, 0.02, 0.5, 3.0])
def test_scales(scale):
    check(*case([600, 40], 10, 2, 6, 14), softmax_scale=scale)


def test_growing_scores_rescale():
    """Scores that rise along the sequence, past what a weight holds without a rescale."""
    q, k, v, t, l, seen = case([1500], 12, 2, 6, 15)
    q[:] = 1.0
    pos = np.arange(1500)
    k[t[0, pos // 16], pos % 16] = (pos / 100.0)[:, None, None].astype(np.float16)
    check(q, k, v, t, l, seen)
    k[t[0, pos // 16], pos % 16] = (-pos / 100.0)[:, None, None].astype(np.float16)
    check(q, k, v, t, l, seen)


def test_strided_q_out_and_pools():
    b, n, h, r = 3, 11, 2, 6
    q, k, v, t, l, seen = case([400, 20, 133], n, h, r, 16)
    wide = torch.zeros(b, n, h * r + 2 * h, 128, dtype=torch.float16, device="cuda")
    qv = wide[:, :, :h * r].unflatten(2, (h, r))
    qv.copy_(dev(q))
    base, _ = check(q, k, v, t, l, seen)
    out = torch.full((b, h, n, r, 128), 3.0, dtype=torch.float16, device="cuda").transpose(1, 2)
    pools = torch.zeros(k.shape[0], 2, h, 16, 128, dtype=torch.float16, device="cuda")
    kp, vp = pools[:, 0].transpose(1, 2), pools[:, 1].transpose(1, 2)
    kp.copy_(dev(k))
    vp.copy_(dev(v))
    words = dev(ref.words_of(seen))
    got = ta().tree_attention(qv, kp, vp, dev(t), dev(l), words, out=out)
    assert got is out and torch.equal(out, base)


def test_repeats_bit_for_bit():
    q, k, v, t, l, seen = (dev(x) for x in case([5000, 300, 2], 20, 2, 6, 17))
    words = dev(ref.words_of(seen.cpu().numpy()))
    a = ta().tree_attention(q, k, v, t, l, words)
    for _ in range(3):
        assert torch.equal(ta().tree_attention(q, k, v, t, l, words), a)


def test_masks_and_depths_of_parents():
    rng = np.random.default_rng(18)
    for n in (1, 2, 63, 64, 65, 130, 256):
        parents = np.stack([ref.random_tree(n, rng, roots) for roots in (1, min(3, n), n)])
        parents[0, n - 1] = n + 5 if n > 1 else -1           # no parent: not before it
        masks, depths = ta().tree_masks(dev(parents))
        seen = np.stack([ref.seen_by(p) for p in parents])
        np.testing.assert_array_equal(masks.cpu().numpy(), ref.words_of(seen))
        np.testing.assert_array_equal(depths.cpu().numpy(), seen.sum(-1) - 1)
