"""Accepted paths and evictions in pools of every order of pages, tokens and heads, on an
MI355X: what contiguous pools come to, bit for bit, and nothing between the rows changed."""

from __future__ import annotations

import itertools

import numpy as np
import pytest

from tests import tree_ref as ref

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]

PAD = 8
ORDERS = list(itertools.permutations(("nb", "t", "h")))


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def stored(values, order):
    """values [nb, 16, H, 128] in a tensor stored as `order` says, rows PAD apart: (view, all)."""
    nb, t, h, d = values.shape
    size = dict(nb=nb, t=t, h=h)
    whole = torch.full((*(size[n] for n in order), d + PAD), 7, dtype=torch.float16, device="cuda")
    view = whole[..., :d].permute(*(order.index(n) for n in ("nb", "t", "h")), 3)
    view.copy_(values)
    return view, whole


def setting(lens, h, layers, seed):
    rng = np.random.default_rng(seed)
    b, width = len(lens), -(-max(lens) // 16) + 1
    nb = b * width + 2
    tables = rng.permutation(nb)[:b * width].reshape(b, width).astype(np.int32)
    pools = rng.integers(-2000, 2000, (2, layers, nb, 16, h, 128)).astype(np.float16)
    return rng, dev(tables), dev(np.array(lens, np.int32)), dev(pools)


def in_every_order(pools, act):
    """act(k_pools, v_pools) of contiguous pools, then of each other order."""
    want = pools.clone()
    first = act(list(want[0]), list(want[1]))
    for order in ORDERS:
        print(f"stored as {order}", flush=True)
        both = [[stored(x, order) for x in side] for side in pools]
        got = act(*([view for view, _ in side] for side in both))
        for a, b in zip(got, first):
            assert torch.equal(a, b)
        for z in (0, 1):
            for li, (view, whole) in enumerate(both[z]):
                assert torch.equal(view, want[z, li])
                assert (whole[..., 128:] == 7).all()
    return first, want


@pytest.mark.parametrize("h,layers", [(1, 1), (3, 2)])
def test_accept(h, layers):
    from latentserve_amd.kernels.hip import tree_attention as ta
    n = 21
    rng, tables, lens, pools = setting([40, n, 77], h, layers, 90 + h)
    parents = np.stack([ref.random_tree(n, rng) for _ in range(3)])
    tokens = rng.integers(0, 3, (3, n)).astype(np.int64)
    choices = rng.integers(0, 3, (3, n)).astype(np.int64)
    for j in range(1, n):
        choices[np.arange(3), parents[:, j]] = tokens[:, j]
    before = pools.clone()
    first, want = in_every_order(pools, lambda k, v: ta.accept_tokens(
        dev(tokens), dev(parents), dev(choices), k, v, tables, lens))
    assert int(first.lengths.max()) > 2 and not torch.equal(want, before)


@pytest.mark.parametrize("h,layers", [(1, 2), (3, 1), (2, 40)])
def test_evict(h, layers):
    from latentserve_amd.kernels.hip import cache_eviction as ce
    rng, tables, lens, pools = setting([700, 40, 333], h, layers, 95 + h)
    sums = dev(rng.random((layers, 3, h, tables.shape[1] * 16)).astype(np.float32))
    before = pools.clone()
    (keep, _), want = in_every_order(pools, lambda k, v: ce.evict_tokens(sums, k, v, tables, lens, 100, 2, 30))
    assert (keep[:, 0, :, 50] > 50).all() and not torch.equal(want, before)
