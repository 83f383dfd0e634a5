"""Pools that accept, move and evict write to: layouts whose rows are apart are taken, in any
order of pages, tokens and heads, and ones whose rows overlap are refused."""

from __future__ import annotations

import itertools

import pytest
import torch

from latentserve_amd import _lib, _tree
from latentserve_amd.kernels.hip import cache_eviction as ce
from latentserve_amd.kernels.hip import tree_attention as ta

NB, H = 5, 3
STORED = dict(nb=NB, t=16, h=H)


def pools(order, pad=0):
    """K and V [nb, 16, H, 128] stored as `order` says, rows `pad` elements longer."""
    def one():
        x = torch.zeros(*(STORED[n] for n in order), 128 + pad, dtype=torch.float16)[..., :128]
        return x.permute(*(order.index(n) for n in ("nb", "t", "h")), 3)
    return one(), one()


def of_strides(*st, h=2, nb=3):
    return [torch.zeros(1 << 16, dtype=torch.float16).as_strided((nb, 16, h, 128), st) for _ in range(2)]


def calls(k, v):
    h = k.shape[2]
    tables, lens = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    one = torch.zeros(1, 1, dtype=torch.int64)
    yield lambda: ta.accept_tokens(one, one.int(), one, [k], [v], tables, lens)
    yield lambda: ce.move_tokens(torch.zeros(1, 1, h, 3, dtype=torch.int32), [k], [v], tables, lens)
    yield lambda: ce.evict_tokens(torch.zeros(1, 1, h, 64), [k], [v], tables, lens, 8)


@pytest.mark.parametrize("pad", [0, 8, 128])
@pytest.mark.parametrize("order", list(itertools.permutations(("nb", "t", "h"))))
def test_rows_that_are_apart_are_taken(order, pad):
    k, v = pools(order, pad)
    h, nb, steps, *_ = _tree.pool_lists([k], [v])
    assert (h, nb, list(steps)) == (H, NB, list(k.stride()[:3]))
    for call in calls(k, v):
        with pytest.raises(ValueError, match="cuda device"):       # (nothing but the device is wrong)
            call()


def test_a_page_that_holds_k_and_v_is_taken():
    both = torch.zeros(NB, 16, 2, H, 128, dtype=torch.float16)
    _tree.pool_lists([both[:, :, 0]], [both[:, :, 1]])
    both = torch.zeros(2, 2, H, 16, 128, dtype=torch.float16)      # one block: its stride does not matter
    _tree.pool_lists([both[:1, 0].transpose(1, 2)], [both[:1, 1].transpose(1, 2)])


@pytest.mark.parametrize("strides,h", [((8192, 256, 256, 1), 2), ((8192, 128, 128, 1), 2), ((4096, 256, 0, 1), 2),
                                       ((4096, 0, 128, 1), 2), ((0, 256, 128, 1), 2), ((4096, 256, 64, 1), 2),
                                       ((128, 384, 128, 1), 2), ((2048, 128, 4096, 1), 2), ((2048, 120, 6144, 1), 2),
                                       ((1024, 128, 4096, 1), 1), ((8192, 256, 1920, 1), 2)])
def test_rows_that_overlap_are_refused(strides, h):
    k, v = of_strides(*strides, h=h)
    for call in calls(k, v):
        with pytest.raises(ValueError, match="overlap"):
            call()


def test_one_head_or_one_block_has_no_stride():
    for strides, h, nb in (((2048, 128, 0, 1), 1, 3), ((0, 256, 128, 1), 2, 1), ((8, 128, 2048, 1), 2, 1)):
        _tree.pool_lists(*([x] for x in of_strides(*strides, h=h, nb=nb)))
