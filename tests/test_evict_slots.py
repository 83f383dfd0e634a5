"""evict() takes slots of the cache only, each once however it is named."""

from __future__ import annotations

import pytest
import torch

from tests.test_bounded_cache import SLOTS, cache, every, grow, held, plain  # noqa: F401


@pytest.mark.parametrize("slots", [[-1, SLOTS - 1], [-1], [SLOTS], [0, SLOTS + 3], [-SLOTS]])
def test_slots_outside_the_cache_are_refused(plain, slots):  # noqa: F811
    c = cache()
    c.enable_weight_sums()
    grow(c, [0, SLOTS - 1], [list(range(50)), list(range(100, 150))])
    before = [list(t.blocks) for t in c.tables], c.weight_sums.clone()
    with pytest.raises(ValueError, match="slot"):
        c.evict(20, slots=slots)
    assert [list(t.blocks) for t in c.tables] == before[0] and torch.equal(c.weight_sums, before[1])
    assert held(c, 0) == every(range(50)) and held(c, SLOTS - 1) == every(range(100, 150))


def test_a_slot_named_twice_is_one(plain):  # noqa: F811
    c = cache()
    c.enable_weight_sums()
    grow(c, [0, 5], [list(range(50)), list(range(100, 150))])
    assert c.evict(20, slots=[5, 0, 5]) == [5, 0]
    assert c.tables[5].dropped == c.tables[0].dropped == 30
