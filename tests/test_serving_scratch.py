"""The counters of captured calls, as bookkeeping on the CPU: two graphs that live never
share a slice, a graph's slices come back when it is gone."""

from __future__ import annotations

import gc

import pytest
import torch

from latentserve_amd import _serving


class Graph:
    """(weakly referable, as torch.cuda.CUDAGraph is)"""


@pytest.fixture
def slabs(monkeypatch):
    """Slabs of 4096 ints on the CPU in place of a GPU's."""
    for name, value in (("_slabs", {}), ("_kept", []), ("_free", {}), ("_SLAB_INTS", 4096)):
        monkeypatch.setattr(_serving, name, value)
    _serving._returned.clear()
    synced = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_serving, "_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", synced.append)

    def room(device):
        have = _serving._slabs.get(device.index)
        if have is None or 2 * have[1] > _serving._SLAB_INTS:
            slab = torch.zeros(_serving._SLAB_INTS, dtype=torch.int32)
            _serving._kept.append(slab)
            _serving._slabs[device.index] = [slab, 0]

    monkeypatch.setattr(_serving, "_room", room)
    return synced


class Dev:
    index, type = 0, "cpu"


def capture(g, sizes):
    with _serving.counters_of(g):
        return [_serving._slice_for_capture(0, n) for n in sizes]


def spans(slices):
    return [(t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in slices]


def apart(slices):
    s = sorted(spans(slices))
    return all(a[1] <= b[0] for a, b in zip(s, s[1:]))


def test_slices_come_back_with_their_graph(slabs):
    sizes, seen = [64, 512, 512, 32, 1000], None
    for _ in range(50):
        g = Graph()
        got = capture(g, sizes)
        assert apart(got) and all(t.numel() % 32 == 0 and t.numel() >= n
                                  for t, n in zip(got, sizes))
        if seen is not None:
            assert sorted(spans(got)) == seen
        seen = sorted(spans(got))
        del g
        gc.collect()
    assert len(_serving._kept) <= 2 and len(slabs) == 49       # (once a capture after a graph's end)


def test_living_graphs_share_nothing(slabs):
    graphs, held = [], []
    for i in range(40):
        g = Graph()
        got = capture(g, [32 * (1 + i % 3), 96])
        graphs.append(g)
        held.append(got)
        if i % 4 == 3:                                   # some end, in any order
            k = (7 * i) % len(graphs)
            del graphs[k], held[k]
            del g
            gc.collect()
        assert apart([t for h in held for t in h])


def test_captures_without_an_owner_keep_theirs(slabs):
    _serving._room(Dev)
    a = _serving._slice_for_capture(0, 64)
    g = Graph()
    b = capture(g, [64])
    del g
    gc.collect()
    c = capture(Graph(), [64])
    assert spans(b) == spans(c) and apart([a] + c)


def test_a_capture_inside_another_ones(slabs):
    one, two = Graph(), Graph()
    with _serving.counters_of(one):
        a = _serving._slice_for_capture(0, 32)
        with _serving.counters_of(two):
            b = _serving._slice_for_capture(0, 32)
        c = _serving._slice_for_capture(0, 32)
    del two
    gc.collect()
    assert [len(s) for _, s in _serving._returned] == [1]
    del one
    gc.collect()
    assert [len(s) for _, s in _serving._returned] == [1, 2] and apart([a, b, c])


def test_a_failed_capture_gives_its_slices_back(slabs):
    g = Graph()
    with pytest.raises(RuntimeError):
        with _serving.counters_of(g):
            a = _serving._slice_for_capture(0, 32)
            raise RuntimeError
    del g
    gc.collect()
    assert spans(capture(Graph(), [32])) == spans([a])


def test_no_slice_left(slabs):
    g = Graph()
    got = capture(g, [2048, 2048, 32])
    assert got[0] is not None and got[1] is not None and got[2] is None


def test_entered_inside_a_capture(slabs, monkeypatch):
    """Nothing that a capture forbids (a synchronisation, a new slab); the slices are listed
    all the same."""
    _serving._room(Dev)
    gone = Graph()
    a = capture(gone, [32])
    del gone
    gc.collect()
    monkeypatch.setattr(_serving, "_capturing", lambda: True)
    monkeypatch.setattr(_serving, "_room", lambda device: pytest.fail("a slab in a capture"))
    g = Graph()
    b = capture(g, [32])
    assert not slabs and apart(a + b)
    del g
    gc.collect()
    assert len(_serving._returned) == 2
