"""accept() ends a step of the sequences that advance() named: where others were made active
since, the device's rows are not theirs, and nothing changes."""

from __future__ import annotations

import pytest
import torch

from tests.test_bounded_cache import cache, every, grow, held, plain  # noqa: F401

TOKENS = torch.tensor([[20, 21, 22], [120, 121, 122]])
PARENTS = torch.tensor([[-1, 0, 1]] * 2, dtype=torch.int32)
CHOICES = torch.tensor([[21, 22, 0], [7, 0, 0]])


@pytest.mark.parametrize("now", [[4], [4, 1], [1, 4, 2], [1, 2]])
def test_other_active_sequences_are_refused(plain, now):  # noqa: F811
    c = cache()
    grow(c, [1, 4, 2], [list(range(14)), list(range(100, 114)), list(range(200, 214))])
    grow(c, [1, 4], TOKENS.tolist())
    c.set_active(now)
    lens = [t.length for t in c.tables]
    with pytest.raises(RuntimeError, match="active"):
        c.accept(TOKENS, PARENTS, CHOICES)
    assert [t.length for t in c.tables] == lens
    assert held(c, 1) == every([*range(14), 20, 21, 22])
    assert held(c, 4) == every([*range(100, 114), 120, 121, 122])
    c.set_active([1, 4])
    c.accept(TOKENS, PARENTS, CHOICES)
    assert held(c, 1) == every([*range(14), 20, 21, 22]) and held(c, 4) == every([*range(100, 114), 120])


def test_a_cache_that_published_anew_goes_on(plain):  # noqa: F811
    """Whatever publishes (compaction, sums enabled) publishes the active sequences."""
    c = cache()
    grow(c, [3], [list(range(40))])
    grow(c, [1, 4], [list(range(14)), list(range(100, 114))])
    grow(c, [1, 4], TOKENS.tolist())
    c.free_sequence(3)
    assert c.compact()
    c.enable_weight_sums()
    c.accept(TOKENS, PARENTS, CHOICES)
    assert c.seq_lens == [17, 15] and held(c, 4) == every([*range(100, 114), 120])
