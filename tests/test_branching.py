"""Forked, rewound, freed and compacted sequences keep their own tokens: the paged
cache's bookkeeping on the CPU, against plain lists."""

from __future__ import annotations

import random

import pytest
import torch

from latentserve_amd.runtime.kv_cache import KVCacheSpec, OutOfBlocks, PagedKVCache
from latentserve_amd.runtime.prefix_cache import PrefixCache

SLOTS, LAYERS, H, D = 6, 2, 1, 8


def cache(blocks=40, max_len=160):
    return PagedKVCache(KVCacheSpec(num_layers=LAYERS, num_kv_heads=H, head_dim=D,
                                    max_batch_size=SLOTS, max_seq_len=max_len, dtype=torch.float32,
                                    device="cpu"), num_blocks=blocks)


def grow(c, slots, tokens):
    """tokens: [len(slots)][n] numbers, written as K (negated as V) of every layer."""
    n = len(tokens[0])
    c.advance(n, slots=slots)
    x = torch.tensor(tokens, dtype=torch.float32).view(len(slots), 1, n, 1).expand(-1, H, -1, D)
    for li in range(LAYERS):
        c.write(li, x + 1000 * li, -x - 1000 * li)


def held(c, slot):
    t = c.tables[slot]
    out = []
    for p in range(t.length):
        s = t.slot(p)
        k = [pool.view(-1, H, D)[s] for pool in c.k_pool]
        v = [pool.view(-1, H, D)[s] for pool in c.v_pool]
        for li in range(LAYERS):
            assert (k[li] == k[0][0, 0] + 1000 * li).all() and (v[li] == -k[li]).all()
        out.append(int(k[0][0, 0]))
    return out


def check(c, want):
    for s in range(SLOTS):
        assert held(c, s) == want[s], s
    refs = [0] * c.num_blocks
    for t in c.tables:
        for b in t.blocks:
            refs[b] += 1
    return refs


def check_refs(c, want, extra=()):
    refs = check(c, want)
    for b in extra:
        refs[b] += 1
    assert refs == [c.allocator.ref_count(b) for b in range(c.num_blocks)]
    assert sorted(c.allocator._stack) == [b for b in range(c.num_blocks) if refs[b] == 0]


def test_branches_share_pages_until_they_write():
    c = cache()
    grow(c, [0], [list(range(20))])
    c.fork(0, [1, 2, 3])
    assert c.allocator.num_used == 2 and c.tables[2].blocks == c.tables[0].blocks
    grow(c, [0, 1, 2], [[100], [101], [102]])
    # slot 3 still holds the first partial page; the writers copied it
    assert c.allocator.num_used == 1 + 4
    assert len({c.tables[s].blocks[1] for s in range(4)}) == 4
    assert len({c.tables[s].blocks[0] for s in range(4)}) == 1
    grow(c, [3], [[103]])                       # the last holder writes in place
    assert c.allocator.num_used == 1 + 4
    base = list(range(20))
    check_refs(c, [base + [100], base + [101], base + [102], base + [103], [], []])


def test_all_branches_writing_at_once_copy_once_less_than_they_are():
    c = cache()
    grow(c, [0], [list(range(5))])
    c.fork(0, [1, 2])
    grow(c, [0, 1, 2], [[7, 8], [9, 10], [11, 12]])
    assert c.allocator.num_used == 3
    check_refs(c, [[0, 1, 2, 3, 4, 7, 8], [0, 1, 2, 3, 4, 9, 10], [0, 1, 2, 3, 4, 11, 12], [], [], []])


def test_fork_at_a_page_border_and_of_nothing():
    c = cache()
    grow(c, [0], [list(range(16))])
    c.fork(0, [1])
    c.fork(4, [5])
    grow(c, [0, 1, 5], [[1], [2], [3]])
    assert c.tables[0].blocks[0] == c.tables[1].blocks[0]
    check_refs(c, [list(range(16)) + [1], list(range(16)) + [2], [], [], [], [3]])


def test_fork_refuses():
    c = cache()
    grow(c, [0, 1], [[1], [2]])
    for children in ([1], [0], [2, 2], [2, 1], [-1], [1000]):
        with pytest.raises(ValueError):
            c.fork(0, children)
    check_refs(c, [[1], [2], [], [], [], []])


def test_no_block_for_a_copy_leaves_everything_as_it_was():
    c = cache(blocks=2)
    grow(c, [0], [list(range(20))])
    c.fork(0, [1])
    with pytest.raises(OutOfBlocks):
        c.advance(1, slots=[0, 1])
    check_refs(c, [list(range(20)), list(range(20)), [], [], [], []])
    c.free_sequence(1)
    grow(c, [0], [[9]])
    check_refs(c, [list(range(20)) + [9], [], [], [], [], []])


def test_a_rewound_branch_does_not_write_the_others_pages():
    c = cache()
    grow(c, [0], [list(range(40))])
    c.fork(0, [1])
    c.rewind(10, slots=[1])
    grow(c, [1], [[70] * 25])
    check_refs(c, [list(range(40)), list(range(10)) + [70] * 25, [], [], [], []])


def test_a_rewound_sequence_does_not_write_a_recorded_prefix_page():
    c = cache()
    p = PrefixCache(c.allocator, 16)
    grow(c, [0], [list(range(33))])
    p.register(list(range(33)), c.tables[0].blocks)
    c.rewind(5, slots=[0])
    grow(c, [0], [[50] * 30])
    got = p.match(list(range(33)))
    assert len(got) == 2
    c.attach_prefix(1, got, 32)
    assert held(c, 1) == list(range(32)) and held(c, 0) == list(range(5)) + [50] * 30
    assert p.num_reclaimable() == p.count_reclaimable_by_scan()


def test_compact_moves_held_pages_down_and_renumbers_every_holder():
    c = cache()
    p = PrefixCache(c.allocator, 16)
    for s in range(4):
        grow(c, [s], [[100 * s + i for i in range(40)]])
    p.register([200 + i for i in range(40)], c.tables[2].blocks)
    c.fork(3, [4])
    c.free_sequence(0)
    c.free_sequence(2)                           # its two whole pages stay recorded
    kept = sorted(p.entry)
    moves = c.compact()
    n = c.allocator.num_used
    assert n == 3 + 3 + 2 and all(old >= n > new for old, new in moves.items())
    want = [[], [100 + i for i in range(40)], [], [300 + i for i in range(40)],
            [300 + i for i in range(40)], []]
    assert sorted(p.entry) == sorted(moves.get(b, b) for b in kept) == sorted(p.lru)
    check_refs(c, want, extra=p.entry)
    got = p.match([200 + i for i in range(40)])
    assert len(got) == 2
    c.attach_prefix(0, got, 32)
    want[0] = [200 + i for i in range(32)]
    check_refs(c, want, extra=p.entry)
    assert c.allocator.allocate(1) == [n]        # the free blocks, lowest first


def test_compact_of_a_compact_or_empty_cache_moves_nothing():
    c = cache()
    assert c.compact() == {}
    grow(c, [0, 1], [[1] * 17, [2] * 17])
    assert c.compact() == {}
    check_refs(c, [[1] * 17, [2] * 17, [], [], [], []])


def test_published_tables_follow_a_compaction():
    c = cache()
    for s in range(3):
        grow(c, [s], [[s] * 30])
    c.set_active([2])
    c.advance(0, slots=[2])
    c.free_sequence(0)
    c.compact()
    row = c.block_tables_tensor(1)[0]
    assert row[:2].tolist() == c.tables[2].blocks


@pytest.mark.parametrize("seed", range(12))
def test_any_sequence_of_steps(seed):
    r = random.Random(seed)
    c = cache(blocks=30, max_len=96)
    p = PrefixCache(c.allocator, 16) if seed % 2 else None
    want, next_token = [[] for _ in range(SLOTS)], 0
    for _ in range(60):
        live = [s for s in range(SLOTS) if want[s]]
        free = [s for s in range(SLOTS) if not want[s]]
        op = r.choice(["grow", "grow", "grow", "fork", "rewind", "free", "compact", "register"])
        try:
            if op == "grow":
                n = r.choice([1, 1, 3, 20])
                slots = [s for s in r.sample(range(SLOTS), r.randint(1, 4))
                         if len(want[s]) + n <= 96]
                if not slots:
                    continue
                lengths = [t.length for t in c.tables]
                toks = [[next_token + i * n + j for j in range(n)] for i in range(len(slots))]
                try:
                    grow(c, slots, toks)
                except OutOfBlocks:
                    # (tables extended before the pool ran out keep their length: put back)
                    for t, k in zip(c.tables, lengths):
                        t.length = k
                    continue
                next_token += n * len(slots)
                for s, t in zip(slots, toks):
                    want[s] = want[s] + t
            elif op == "fork" and live and free:
                s, kids = r.choice(live), r.sample(free, r.randint(1, len(free)))
                kids = [k for k in kids if not c.tables[k].blocks]
                c.fork(s, kids)
                for k in kids:
                    want[k] = list(want[s])
            elif op == "rewind" and live:
                s = r.choice(live)
                n = r.randint(1, len(want[s]))
                c.rewind(n, slots=[s])
                want[s] = want[s][:n]
            elif op == "free" and live:
                s = r.choice(live)
                c.free_sequence(s)
                want[s] = []
            elif op == "compact":
                c.compact()
                held_blocks = [b for b in range(c.num_blocks) if c.allocator.ref_count(b)]
                assert held_blocks == list(range(c.allocator.num_used))
            elif op == "register" and p and live:
                s = r.choice(live)
                p.register(want[s], c.tables[s].blocks)
        finally:
            check_refs(c, want, extra=p.entry if p else ())
            if p:
                assert p.num_reclaimable() == p.count_reclaimable_by_scan()
