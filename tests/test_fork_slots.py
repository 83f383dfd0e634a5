"""fork() takes slots of the cache only, the forked one included, on every paged cache."""

from __future__ import annotations

import pytest
import torch

from latentserve_amd.runtime.int4_cache import Int4PagedKVCache
from latentserve_amd.runtime.int8_cache import Int8PagedKVCache
from latentserve_amd.runtime.kv_cache import KVCacheSpec, PagedKVCache


@pytest.mark.parametrize("kind", [PagedKVCache, Int8PagedKVCache, Int4PagedKVCache])
@pytest.mark.parametrize("index,children", [(-1, [1]), (-4, [1]), (4, [1]), (100, []), (2, [2]),
                                            (2, [1, 2]), (0, [4]), (0, [-2])])
def test_fork_of_a_slot_that_is_none_or_its_own_child(kind, index, children):
    c = kind(KVCacheSpec(num_layers=1, num_kv_heads=1, head_dim=128, max_batch_size=4,
                         max_seq_len=64, dtype=torch.float16, device="cpu"))
    c.advance(5, slots=[0, 3])
    before = [(list(t.blocks), t.length, t.version) for t in c.tables]
    refs = list(c.allocator._refs)
    with pytest.raises(ValueError):
        c.fork(index, children)
    assert before == [(t.blocks, t.length, t.version) for t in c.tables]
    assert refs == c.allocator._refs
    c.fork(3, [1, 2])
    assert c.tables[1].blocks == c.tables[3].blocks and c.tables[2].length == 5
