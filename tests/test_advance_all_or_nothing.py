"""A step that the pool cannot hold leaves the cache as it was: advance() of the paged
caches on the CPU, with branches, a prefix cache and steps that run out of blocks."""

from __future__ import annotations

import copy
import random

import pytest
import torch

from latentserve_amd.runtime.int4_cache import Int4PagedKVCache
from latentserve_amd.runtime.int8_cache import Int8PagedKVCache
from latentserve_amd.runtime.kv_cache import KVCacheSpec, OutOfBlocks, PagedKVCache
from latentserve_amd.runtime.prefix_cache import PrefixCache
from tests.test_branching import SLOTS, cache, check_refs, grow, held

CACHES = [PagedKVCache, Int8PagedKVCache, Int4PagedKVCache]


def of(kind, blocks, max_len=160):
    return kind(KVCacheSpec(num_layers=2, num_kv_heads=1, head_dim=128, max_batch_size=SLOTS,
                            max_seq_len=max_len, dtype=torch.float16, device="cpu"),
                num_blocks=blocks)


def state(c):
    return copy.deepcopy(([(t.blocks, t.length) for t in c.tables], c._active, c.allocator._refs,
                          sorted(c.allocator._stack), c.inputs.tables, c.inputs.vec["lens"],
                          getattr(c, "_pooled", None)))


def same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y, (x, y)


@pytest.mark.parametrize("kind", CACHES)
def test_a_copy_and_a_page_too_many(kind):
    """One block is left; the step needs it for a private copy, and one more for the third
    sequence's next page."""
    c = of(kind, 4)
    c.advance(20, slots=[0])
    c.advance(16, slots=[2])
    c.fork(0, [1])
    before = state(c)
    for _ in range(3):
        with pytest.raises(OutOfBlocks):
            c.advance(1, slots=[0, 1, 2])
        same(state(c), before)
    assert c.active_slots == [2]
    c.free_sequence(2)
    c.advance(1, slots=[0, 1])
    assert [c.tables[s].length for s in range(3)] == [21, 21, 0]
    assert c.tables[0].blocks[1] != c.tables[1].blocks[1]


@pytest.mark.parametrize("kind", CACHES)
def test_a_later_sequence_without_a_page(kind):
    c = of(kind, 5)
    c.advance(30, slots=[0, 1])
    before = state(c)
    with pytest.raises(OutOfBlocks):
        c.advance(3, slots=[0, 1])
    same(state(c), before)
    c.advance(2, slots=[0, 1])
    assert [c.tables[s].length for s in range(2)] == [32, 32]


@pytest.mark.parametrize("kind", CACHES)
def test_a_sequence_past_the_capacity(kind):
    c = of(kind, 40, max_len=32)
    c.advance(20, slots=[0, 1])
    before = state(c)
    with pytest.raises(RuntimeError, match="sized for 2"):
        c.advance(13, slots=[0, 1])
    same(state(c), before)
    c.advance(12, slots=[0, 1])


@pytest.mark.parametrize("kind", CACHES)
def test_a_sequence_named_twice_is_refused(kind):
    c = of(kind, 20)
    c.advance(5, slots=[0, 1])
    before = state(c)
    for slots in ([0, 0], [1, 0, 1]):
        with pytest.raises(ValueError):
            c.advance(1, slots=slots)
        same(state(c), before)


def test_a_page_of_bounds_owned_once_where_a_rewind_names_a_sequence_twice(monkeypatch):
    c = cache()
    grow(c, [0], [list(range(20))])
    c.fork(0, [1, 2])
    c.kmin = c.kmax = []                             # (page bounds are the GPU's to keep)
    monkeypatch.setattr(c, "_bound_partial_page", lambda *a: None)
    c.rewind(18, slots=[1, 1])
    base = list(range(20))
    check_refs(c, [base, base[:18], base, [], [], []])


@pytest.mark.parametrize("kind", CACHES)
def test_a_step_of_no_tokens_copies_no_page(kind):
    """advance(0) publishes the sequences; their shared pages stay shared, and no block is
    asked for."""
    c = of(kind, 2)
    c.advance(20, slots=[0])
    c.fork(0, [1, 2])
    c.advance(0, slots=[0, 2])
    assert c.allocator.num_used == 2 and c.active_slots == [0, 2]
    assert c.tables[0].blocks == c.tables[1].blocks == c.tables[2].blocks
    assert c.seq_lens_tensor(2).tolist() == [20, 20]
    assert c.block_tables_tensor(2)[:, :2].tolist() == [c.tables[0].blocks] * 2


def test_blocks_that_a_prefix_cache_holds_alone_count():
    """A step takes what reclaiming gives, copies and pages together; one more is too many."""
    for blocks, fits in ((6, True), (5, False)):
        c = cache(blocks=blocks)
        p = PrefixCache(c.allocator, 16)
        grow(c, [5], [[900 + i for i in range(32)]])
        p.register([900 + i for i in range(32)], c.tables[5].blocks)
        c.free_sequence(5)                           # two pages the prefix cache holds alone
        grow(c, [0], [list(range(20))])
        c.fork(0, [1])
        grow(c, [2], [[50] * 16])
        want = [list(range(20)), list(range(20)), [50] * 16, [], [], []]
        check_refs(c, want, extra=p.entry)
        if fits:
            grow(c, [0, 1, 2], [[1], [2], [3]])
            want = [w + [i + 1] for i, w in enumerate(want[:3])] + [[], [], []]
        else:
            grow(c, [3], [[60] * 16])                # takes a recorded page
            want[3] = [60] * 16
            with pytest.raises(OutOfBlocks):
                grow(c, [0, 1, 2], [[1], [2], [3]])
        check_refs(c, want, extra=p.entry)
        assert p.num_reclaimable() == p.count_reclaimable_by_scan()


@pytest.mark.parametrize("seed", range(16))
def test_steps_that_run_out_of_blocks_change_nothing(seed):
    r = random.Random(100 + seed)
    c = cache(blocks=14, max_len=96)
    p = PrefixCache(c.allocator, 16) if seed % 2 else None
    want, token, failed = [[] for _ in range(SLOTS)], 0, 0
    for _ in range(80):
        live = [s for s in range(SLOTS) if want[s]]
        free = [s for s in range(SLOTS) if not want[s] and not c.tables[s].blocks]
        op = r.choice(["grow"] * 5 + ["fork", "rewind", "free", "compact", "register"])
        if op == "grow":
            n = r.choice([1, 1, 3, 20])
            slots = [s for s in r.sample(range(SLOTS), r.randint(1, 5)) if len(want[s]) + n <= 96]
            toks = [[token + i * n + j for j in range(n)] for i in range(len(slots))]
            if slots:
                tables, active = [(list(t.blocks), t.length) for t in c.tables], c.active_slots
                try:
                    grow(c, slots, toks)
                    token += n * len(slots)
                    for s, t in zip(slots, toks):
                        want[s] = want[s] + t
                except OutOfBlocks:
                    failed += 1
                    assert tables == [(t.blocks, t.length) for t in c.tables]
                    assert active == c.active_slots
        elif op == "fork" and live and free:
            s, kids = r.choice(live), r.sample(free, r.randint(1, len(free)))
            c.fork(s, kids)
            for k in kids:
                want[k] = list(want[s])
        elif op == "rewind" and live:
            s = r.choice(live)
            n = r.randint(1, len(want[s]))
            c.rewind(n, slots=[s])
            want[s] = want[s][:n]
        elif op == "free" and live and r.random() < 0.5:
            s = r.choice(live)
            c.free_sequence(s)
            want[s] = []
        elif op == "compact":
            c.compact()
        elif op == "register" and p and live:
            s = r.choice(live)
            p.register(want[s], c.tables[s].blocks)
        check_refs(c, want, extra=p.entry if p else ())
        if p:
            assert p.num_reclaimable() == p.count_reclaimable_by_scan()
    assert failed and [held(c, s) for s in range(SLOTS)] == want
