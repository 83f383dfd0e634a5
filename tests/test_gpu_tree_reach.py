"""The drafted-tree and eviction operators where addresses and lists get long, on an
MI355X: pools past 4 GiB, strided pools, moves of many rounds and many lists, graphs of
acceptances and evictions.  A call's bits follow from what it reads alone, so the far or
strided call is held to the same call on small contiguous pools."""

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


def ta():
    from latentserve_amd.kernels.hip import tree_attention
    return tree_attention


def ce():
    from latentserve_amd.kernels.hip import cache_eviction
    return cache_eviction


def everything(q, k, v, tables, lens, words, budget=200):
    """Each operator once, on the pools it is given; what they return and leave."""
    b, n, h, r, _ = q.shape
    lse = torch.zeros(b, n, h, r, device="cuda")
    width = tables.shape[1] * 16
    print(f"everything {tuple(q.shape)} pool {tuple(k.shape)} {k.stride()}", flush=True)
    out = ta().tree_attention(q, k, v, tables, lens, words, lse=lse)
    rng = np.random.default_rng(1)
    tokens = dev(rng.integers(0, 2, (b, n)))
    parents = dev(np.stack([ref.random_tree(n, rng) for _ in range(b)]))
    choices = dev(rng.integers(0, 2, (b, n)))
    got = ta().accept_tokens(tokens, parents, choices, [k], [v], tables, lens)
    left = (lens - n).clamp(min=0) + got.lengths
    sums = torch.zeros(b, h, width, device="cuda")
    ce().add_weights(q, lse, k, tables, left, sums, path=got.path, lengths=got.lengths)
    one = ce().paged_decode_weights(q[:, 0].contiguous(), k, v, tables, left, sums)
    keep, kept = ce().evict_tokens(sums[None], [k], [v], tables, left, budget)
    again = ta().tree_attention(q[:, :1], k, v, tables, left.clamp(max=budget))
    torch.cuda.synchronize()
    return out, lse, *got, sums, one, keep, kept, again


@pytest.mark.parametrize("n,r", [(2, 6), (5, 6), (16, 4), (33, 6)])
def test_pools_past_four_gigabytes(n, r):
    q, k, v, t, l, seen = case([900, 333, n], n, 8, r, 90 + n)
    want = everything(dev(q), dev(k), dev(v), dev(t), dev(l), dev(ref.words_of(seen)))
    nb = 140000                                              # of 32 KiB: 4.6 GB a pool
    ids = np.random.default_rng(2).permutation(nb - 66000)[:k.shape[0]] + 66000
    far = [torch.empty(nb, 16, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    for pool, x in zip(far, (k, v)):
        pool[0] = 0
        pool[dev(ids)] = dev(x)
    got = everything(dev(q), *far, dev(ids[t].astype(np.int32)), dev(l), dev(ref.words_of(seen)))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,r", [(3, 6), (12, 6), (40, 4)])
def test_strided_pools(n, r):
    q, k, v, t, l, seen = case([500, 120, n + 1], n, 2, r, 95 + n)
    want = everything(dev(q), dk := dev(k), dv := dev(v), dev(t), dev(l), dev(ref.words_of(seen)))
    # heads 1 and 3 of five, of every second block, rows longer than they need
    big = [torch.full((2 * k.shape[0], 16, 5, 136), 7.0, dtype=torch.float16, device="cuda")
           for _ in range(2)]
    views = [x[1::2, :, 1:4:2, :128] for x in big]
    for view, x in zip(views, (k, v)):
        view.copy_(dev(x))
    got = everything(dev(q), *views, dev(t), dev(l), dev(ref.words_of(seen)))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for x, view, y in zip(big, views, (dk, dv)):
        assert torch.equal(view, y)
        view.fill_(7.0)
        assert (x == 7.0).all()                              # nothing beside the rows was touched


@pytest.mark.parametrize("lens,budget,h,layers", [([1500, 40, 1101], 1100, 2, 12),     # 144 lists
                                                  ([9000], 5000, 1, 1), ([2047, 2049], 1024, 3, 1),
                                                  ([33, 40] * 40, 31, 1, 1)])
def test_moves_of_many_rounds_and_lists(lens, budget, h, layers):
    rng = np.random.default_rng(54)
    b = len(lens)
    width = -(-max(lens) // 16)
    nb = b * width + 1
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    pools = torch.randint(-2000, 2000, (2, layers, nb, 16, h, 128), device="cuda",
                          generator=torch.Generator("cuda").manual_seed(3)).half()
    keep = np.full((layers, b, h, budget), -1, np.int32)
    for x in range(layers):
        for i, n in enumerate(lens):
            for y in range(h):
                m = min(n, budget)
                keep[x, i, y, :m] = np.sort(rng.permutation(n)[:m])
    want = pools.clone()
    for x in range(layers):
        for i, n in enumerate(lens):
            for y in range(h):
                src = keep[x, i, y, :min(n, budget)]
                dst = np.arange(len(src))
                at = [dev(z.astype(np.int64)) for z in (tables[i, dst // 16], dst % 16,
                                                        tables[i, src // 16], src % 16)]
                want[:, x, at[0], at[1], y] = pools[:, x, at[2], at[3], y]
    print(f"move {lens[:4]} {budget} h={h} layers={layers}", flush=True)
    ce().move_tokens(dev(keep), list(pools[0]), list(pools[1]), dev(tables),
                     dev(np.array(lens, np.int32)))
    assert torch.equal(pools, want)


def test_graphs_of_acceptance_and_eviction():
    """A step and an eviction captured, replayed from the same pools with eager work between."""
    n = 6
    q, k, v, t, l, seen = case([700, 90, n], n, 2, 6, 71)
    args = [dev(x) for x in (q, k, v, t, l)]
    words = dev(ref.words_of(seen))
    first = [x.clone() for x in args[1:3]]
    rng = np.random.default_rng(1)
    tokens = dev(rng.integers(0, 2, (3, n)))
    parents = dev(np.stack([ref.random_tree(n, rng) for _ in range(3)]))
    choices = dev(rng.integers(0, 2, (3, n)))

    def step():
        q_, k_, v_, t_, l_ = args
        lse = torch.zeros(3, n, 2, 6, device="cuda")
        out = ta().tree_attention(q_, k_, v_, t_, l_, words, lse=lse)
        got = ta().accept_tokens(tokens, parents, choices, [k_], [v_], t_, l_)
        left = (l_ - n).clamp(min=0) + got.lengths
        sums = torch.zeros(3, 2, t.shape[1] * 16, device="cuda")
        ce().add_weights(q_, lse, k_, t_, left, sums, path=got.path, lengths=got.lengths)
        one = ce().paged_decode_weights(q_[:, 0].contiguous(), k_, v_, t_, left, sums)
        keep, kept = ce().evict_tokens(sums[None], [k_], [v_], t_, left, 64)
        return out, lse, *got, sums, one, keep, kept

    def again():
        for x, y in zip(args[1:3], first):
            x.copy_(y)

    want = [x.clone() for x in step()] + [x.clone() for x in args[1:3]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = step()
        graphs.append((g, outs))
    for turn in range(3):
        for g, outs in graphs:
            again()
            print(f"replay {turn}", flush=True)
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip([*outs, *args[1:3]], want):
                assert torch.equal(x, y)
            again()
            for x, y in zip([*step(), *args[1:3]], want):
                assert torch.equal(x, y)


@pytest.mark.parametrize("lens", [[300, 256, 20], [1500]])
def test_the_largest_trees(lens):
    from tests.test_gpu_tree_attention import check
    check(*case(lens, 256, 1, 16, 98))


@pytest.mark.parametrize("b,h,r", [(300, 4, 6), (70, 1, 16), (65, 8, 1)])
def test_decode_weights_of_many_sequences(b, h, r):
    """More sequences than are dealt whole, some without a token."""
    lens = [(37 * i) % 90 for i in range(b)]
    q, k, v, t, l, _ = case(lens, 1, h, r, 99)
    sums = torch.zeros(b, h, t.shape[1] * 16, device="cuda")
    print(f"decode weights of {b}", flush=True)
    out = ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), sums)
    want, lse, tol, _ = ref.attend(q, k, v, t, l)
    assert (np.abs(out.double().cpu().numpy() - want[:, 0]) <= tol[:, 0]).all()
    add, atol = ref.path_weights(q, lse, k, t, l, np.zeros((b, 1), np.int32), np.ones(b, np.int32))
    n = add.shape[2]
    got = sums.double().cpu().numpy()
    assert (np.abs(got[..., :n] - add) <= 2 * atol + add * 2.0 ** -16).all()
    assert (got[..., n:] == 0).all()


def test_a_longer_batch_leaves_rows_behind_the_last_sequence():
    """out and lse of a larger buffer, pools' unused pages and the sums' other rows stay."""
    q, k, v, t, l, seen = case([70, 33], 5, 2, 6, 100)
    big = torch.full((4, 5, 2, 6, 128), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((4, 5, 2, 6), 7.0, device="cuda")
    ta().tree_attention(dev(q), dev(k), dev(v), dev(t), dev(l), dev(ref.words_of(seen)),
                        out=big[:2], lse=lse[:2])
    assert (big[2:] == 7).all() and (lse[2:] == 7).all() and not (big[:2] == 7).all()
    sums = torch.full((5, 2, 100), 3.0, device="cuda")
    rows = dev(np.array([4, 1], np.int32))
    ce().paged_decode_weights(dev(q[:, 0]), dev(k), dev(v), dev(t), dev(l), sums, rows)
    assert (sums[[0, 2, 3]] == 3).all() and (sums[4, :, 70:] == 3).all() and (sums[1, :, 33:] == 3).all()
    assert (sums[4, :, :70] > 3).all()
