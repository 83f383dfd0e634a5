"""Batches of none, sums of no rows and of no tokens, on an MI355X."""

from __future__ import annotations

import pytest

from tests.test_gpu_tree_attention import case, dev

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def test_masks_of_no_trees():
    from latentserve_amd.kernels.hip.tree_attention import tree_masks
    masks, depths = tree_masks(torch.empty(0, 70, dtype=torch.int32, device="cuda"))
    assert masks.shape == (0, 70, 2) and depths.shape == (0, 70)


@pytest.mark.parametrize("rows,length", [(3, 0), (0, 64), (0, 0)])
def test_sums_of_nothing(rows, length):
    from latentserve_amd.kernels.hip import cache_eviction as ce
    q, k, v, t, l, _ = case([200, 33], 1, 2, 6, 77)
    dq, dk, dv, dt, dl = (dev(x) for x in (q, k, v, t, l))
    q1 = dq[:, 0].contiguous()
    want = ce.paged_decode_weights(q1, dk, dv, dt, dl, torch.zeros(2, 2, 208, device="cuda"))
    sums = torch.empty(rows, 2, length, device="cuda")
    of = torch.zeros(2, dtype=torch.int32, device="cuda")
    of[1] = 1
    got = ce.paged_decode_weights(q1, dk, dv, dt, dl, sums, of)
    assert torch.equal(got, want)
    ce.add_weights(dq, torch.ones(2, 1, 2, 6, device="cuda"), dk, dt, dl, sums, of)
    torch.cuda.synchronize()


def test_selection_from_no_tokens():
    from latentserve_amd.kernels.hip import cache_eviction as ce
    lens = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    keep, kept = ce.select_tokens(torch.empty(3, 2, 2, 0, device="cuda"), lens, 4, 1, 1)
    assert (keep == -1).all() and (kept == 0).all()
