"""Rewinding a sequence that lost tokens to a budget: to nothing, to rows that all heads
share, and to rows that they do not (refused), on the CPU."""

from __future__ import annotations

import pytest
import torch

from tests.test_bounded_cache import cache, every, grow, held, plain, sums_for  # noqa: F401


def bounded(c, slot=0, tokens=90, budget=20, sinks=2, recent=5, first=0):
    grow(c, [slot], [list(range(first, first + tokens))])
    sums_for(c, slot, [[[7, 30], [8, 31]], [[9, 32], [10, 33]]])
    c.evict(budget, sinks=sinks, recent=recent, slots=[slot])


def state(c):
    return ([list(t.blocks) for t in c.tables], [(t.length, t.dropped) for t in c.tables],
            c.weight_sums.clone(), c.active_slots, c.seq_lens_tensor().tolist())


def unchanged(c, before):
    return all(torch.equal(a, b) if torch.is_tensor(a) else a == b for a, b in zip(state(c), before))


def test_a_rewind_to_nothing_starts_anew(plain):  # noqa: F811
    c = cache()
    c.max_positions = 100
    c.enable_weight_sums()
    bounded(c)
    assert c.seq_positions == [90]
    c.rewind(0, slots=[0])
    assert c.seq_positions == [0] and c.tables[0].dropped == 0
    assert (c.weight_sums[:, 0] == 0).all()
    grow(c, [0], [list(range(30))])
    assert c.seq_positions == [30] and held(c, 0) == every(range(30))
    assert c.shareable_blocks(0) == 1
    grow(c, [0], [list(range(30, 130))])                   # (no bound but the capacity)
    assert c.seq_positions == [130]


@pytest.mark.parametrize("length", [1, 2, 3, 10, 14])
def test_a_rewind_among_rows_that_differ_by_head_is_refused(plain, length):  # noqa: F811
    c = cache()
    c.enable_weight_sums()
    bounded(c)
    grow(c, [1], [list(range(40))])
    c.set_active([1, 0])
    c.advance(0, slots=[1, 0])
    before = state(c)
    with pytest.raises(ValueError, match="evicted"):
        c.rewind(length, slots=[1, 0])
    assert unchanged(c, before)
    assert len({tuple(x) for layer in held(c, 0) for x in layer}) > 1


def test_a_rewind_of_the_recent_tokens(plain):  # noqa: F811
    c = cache()
    c.enable_weight_sums()
    bounded(c)
    c.rewind(15, slots=[0])                                # the boundary: 20 - 5
    assert c.seq_positions == [85]
    grow(c, [0], [[500, 501]])
    assert c.seq_positions == [87]
    for layer in held(c, 0):
        for x in layer:
            assert x[:2] == [0, 1] and x[15:] == [500, 501]


def test_a_second_eviction_and_forks_keep_the_bound(plain):  # noqa: F811
    c = cache()
    c.enable_weight_sums()
    bounded(c)                                             # 20 held, rows of all heads from 15
    c.fork(0, [3])
    grow(c, [0], [[90, 91, 92]])
    c.evict(21, sinks=0, recent=21, slots=[0])             # two rows off the front: from 13
    assert c.seq_positions == [93]
    before = state(c)
    with pytest.raises(ValueError, match="evicted"):
        c.rewind(12, slots=[0])
    assert unchanged(c, before)
    c.rewind(13, slots=[0])
    assert c.seq_positions == [85]
    c.set_active([3])
    c.advance(0, slots=[3])
    with pytest.raises(ValueError, match="evicted"):
        c.rewind(14)
    c.rewind(15)
    assert c.seq_positions == [85]
    c.free_sequence(3)
    grow(c, [3], [list(range(40))])
    c.rewind(1)
    assert c.seq_positions == [1] and held(c, 3) == every([0])


def test_an_acceptance_ends_behind_the_evicted_rows(plain):  # noqa: F811
    """Drafted tokens are the ones that advance() added: rows that heads do not share are none."""
    c = cache()
    c.enable_weight_sums()
    bounded(c)
    before = state(c)
    tokens = torch.arange(8)[None]
    parents = torch.arange(-1, 7, dtype=torch.int32)[None]
    with pytest.raises(ValueError, match="drafted"):
        c.accept(tokens, parents, tokens)
    assert unchanged(c, before)
