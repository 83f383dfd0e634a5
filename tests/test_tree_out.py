"""An `out` whose own rows overlap is refused by the tree attention and by the decode that
sums weights (two rows' results would race); a strided one is taken.  On the CPU."""

from __future__ import annotations

import itertools

import pytest
import torch

from latentserve_amd.kernels.hip import cache_eviction as ce
from latentserve_amd.kernels.hip import tree_attention as ta

B, N, H, R = 2, 3, 2, 6
HALF = torch.float16


def calls(out):
    """Both entry points with outs of the shape [B, N, H, R, 128] and [B, H, R, 128]."""
    k = torch.zeros(9, 16, H, 128, dtype=HALF)
    t, l = torch.zeros(B, 4, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    q = torch.zeros(B, N, H, R, 128, dtype=HALF)
    if out.dim() == 5:
        ta.tree_attention(q, k, k.clone(), t, l, out=out)
    else:
        ce.paged_decode_weights(q[:, 0], k, k.clone(), t, l, torch.zeros(B, H, 64), out=out)


@pytest.mark.parametrize("dims", [(B, N, H, R), (B, H, R)])
def test_rows_over_each_other_are_refused(dims):
    base = torch.zeros(*dims, 128, dtype=HALF)
    for i in range(len(dims)):
        out = base.narrow(i, 0, 1).expand(*dims, 128)
        with pytest.raises(ValueError, match="out.*overlap"):
            calls(out)
    *st, one = base.stride()
    flat = torch.zeros(1 << 17, dtype=HALF)
    for bad in ([*st[:-1], 64, one], [*st[:-2], st[-1] * (R - 1), st[-1], one]):
        with pytest.raises(ValueError, match="out.*overlap"):
            calls(flat.as_strided((*dims, 128), bad))


@pytest.mark.parametrize("dims", [(B, N, H, R), (B, H, R)])
def test_rows_that_are_apart_are_taken(dims):
    n = len(dims)
    outs = [torch.zeros(*dims, 136, dtype=HALF)[..., :128],
            torch.zeros(dims[0], 2 * dims[1], *dims[2:], 128, dtype=HALF)[:, ::2]]
    for order in itertools.permutations(range(n)):
        x = torch.zeros(*(dims[i] for i in order), 128, dtype=HALF)
        outs.append(x.permute(*(order.index(i) for i in range(n)), n))
    for out in outs:
        with pytest.raises(ValueError, match="cuda device"):       # (nothing but the device is wrong)
            calls(out)
