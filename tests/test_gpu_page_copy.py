"""Page copies against indexing, bit for bit, on an MI355X."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def copy(*a):
    from latentserve_amd.kernels.hip import page_copy
    return page_copy.copy_pages(*a)


def tensors(nb, shapes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, 256, (nb, n), generator=g, device="cuda", dtype=torch.uint8)
            for n in shapes]


@pytest.mark.parametrize("shapes", [[4096], [1], [3], [6, 10], [8192, 8192, 128, 64], [100000],
                                    [4096] * 70, [16 * i + 16 for i in range(65)]],
                         ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("pairs", [1, 7, 200])
def test_copy_is_indexing(shapes, pairs):
    nb = 2 * pairs + 3
    ids = np.random.default_rng(pairs).permutation(nb).tolist()
    src, dst = ids[:pairs], ids[pairs:2 * pairs]
    ts = tensors(nb, shapes)
    want = [t.clone() for t in ts]
    for w in want:
        w[dst] = w[src]
    print(f"copy {len(shapes)} tensors, {pairs} pairs", flush=True)
    copy(ts, src, dst)
    for t, w in zip(ts, want):
        assert torch.equal(t, w)


def test_one_page_to_many_and_numpy_numbers():
    t = torch.randn(300, 16, 2, 128, device="cuda").half()
    w = t.clone()
    dst = np.arange(10, 290)
    w[10:290] = w[5]
    copy([t], np.full(280, 5), dst)
    assert torch.equal(t, w)


def test_types_strides_offsets_and_empty_lists():
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(9, 3, 16, 64, generator=g, device="cuda")
    parts = [wide[:, 1], torch.arange(9 * 5, device="cuda").view(9, 5),
             torch.randn(40, 7, generator=g, device="cuda").half()[1:10],
             torch.zeros(9, 0, device="cuda")]
    want = [p.clone() for p in parts]
    for w in want:
        w[[7, 0]] = w[[2, 3]]
    outside = wide[:, [0, 2]].clone()
    copy(parts, [2, 3], [7, 0])
    for p, w in zip(parts, want):
        assert torch.equal(p, w)
    assert torch.equal(wide[:, [0, 2]], outside)
    copy(parts, [], [])
    copy([], [1], [2])
    for p, w in zip(parts, want):
        assert torch.equal(p, w)


def test_refused_calls_copy_nothing():
    t = torch.arange(20, device="cuda").view(10, 2)
    w = t.clone()
    for src, dst in (([0], [10]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1 << 32]),
                     ([0.5], [1]), (torch.tensor([0], device="cuda"), [1])):
        with pytest.raises(ValueError):
            copy([t], src, dst)
    with pytest.raises(ValueError):
        copy([t, t.cpu()], [0], [1])
    with pytest.raises(ValueError):
        copy([t[:, :0]], [0], [10])
    with pytest.raises(ValueError):
        copy([t[:0]], [0], [1])
    torch.cuda.synchronize()
    assert torch.equal(t, w)


def test_pages_past_32_bit_offsets():
    t = torch.empty(5, 1 << 30, dtype=torch.uint8, device="cuda")
    t[0].fill_(3), t[4].fill_(9)
    copy([t], [4], [1])
    assert (t[1, ::4097] == 9).all() and t[1, -1] == 9 and (t[0, ::4097] == 3).all()


def test_captured_copy_replays():
    ts = tensors(12, [4096, 48])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        copy(ts, [1, 2], [5, 6])
    for rep in range(3):
        for t in ts:
            t[1:3] += 17
        want = [t.clone() for t in ts]
        for w in want:
            w[[5, 6]] = w[[1, 2]]
        g.replay()
        torch.cuda.synchronize()
        for t, w in zip(ts, want):
            assert torch.equal(t, w), rep
