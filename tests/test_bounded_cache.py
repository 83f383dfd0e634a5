"""Accepting drafted trees and evicting to a budget: the paged cache's bookkeeping on the
CPU, with plain forms of the operators in the kernels' place."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from latentserve_amd.kernels.hip import cache_eviction as ce
from latentserve_amd.kernels.hip import tree_attention as ta
from latentserve_amd.runtime.kv_cache import KVCacheSpec, OutOfBlocks, PagedKVCache
from latentserve_amd.runtime.prefix_cache import PrefixCache

SLOTS, LAYERS, H, D = 6, 2, 2, 8


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
    """[layers][heads] lists of a slot's numbers, K and V alike."""
    t = c.tables[slot]
    at = [t.slot(p) for p in range(t.length)]
    out = []
    for li in range(LAYERS):
        k, v = (pool[li].view(-1, H, D)[at] for pool in (c.k_pool, c.v_pool))
        assert torch.equal(v, -k) and (k == k[..., :1]).all()
        out.append([(k[:, h, 0] - 1000 * li).int().tolist() for h in range(H)])
    return out


def every(numbers):
    return [[list(numbers)] * H] * LAYERS


def place(tables, b, p):
    return int(tables[b, p // 16]) * 16 + p % 16


def plain_evict(sums, k_pools, v_pools, tables, lens, budget, sinks, recent):
    layers, b, h, _ = sums.shape
    keep = torch.full((layers, b, h, budget), -1, dtype=torch.int32)
    kept = torch.zeros(layers, b, h, budget)
    for l in range(layers):
        for s in range(b):
            n = int(lens[s])
            for hh in range(h):
                x = sums[l, s, hh, :n].clone()
                x[:sinks] = np.inf
                x[n - recent:] = np.inf
                at = torch.sort(torch.sort(x, descending=True, stable=True)[1][:budget])[0]
                keep[l, s, hh, :len(at)] = at.int()
                kept[l, s, hh, :len(at)] = sums[l, s, hh][at]
                for pool in (k_pools[l], v_pools[l]):
                    rows = pool.view(-1, h, pool.shape[-1])
                    new = rows[[place(tables, s, int(p)) for p in at], hh]
                    rows[[place(tables, s, p) for p in range(len(at))], hh] = new
    return keep, kept


def plain_accept(tokens, parents, choices, k_pools, v_pools, tables, lens, counts=None):
    b, n = tokens.shape
    path = torch.full((b, n), -1, dtype=torch.int32)
    lengths, nxt = torch.zeros(b, dtype=torch.int32), torch.full((b,), -1)
    for s in range(b):
        nodes, at, got = n if counts is None else int(counts[s]), 0, []
        while at is not None and at < nodes:
            got.append(at)
            at = next((j for j in range(at + 1, nodes) if parents[s, j] == at
                       and tokens[s, j] == choices[s, at]), None)
        path[s, :len(got)] = torch.tensor(got, dtype=torch.int32)
        lengths[s] = len(got)
        if got:
            nxt[s] = choices[s, got[-1]]
        base = int(lens[s]) - n
        for pool in (*k_pools, *v_pools):
            rows = pool.view(-1, *pool.shape[2:])
            rows[[place(tables, s, base + i) for i in range(len(got))]] = \
                rows[[place(tables, s, base + i) for i in got]]
    return ta.AcceptedTokens(path, lengths, nxt)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(ce, "evict_tokens", plain_evict)
    monkeypatch.setattr(ta, "accept_tokens", plain_accept)


def test_accept_keeps_the_path_and_shortens_the_sequence(plain):
    c = cache()
    grow(c, [1, 4], [list(range(14)), list(range(100, 114))])
    grow(c, [1, 4], [[20, 21, 22, 23, 24], [120, 121, 122, 123, 124]])
    tokens = torch.tensor([[20, 21, 22, 23, 24]] * 2)
    parents = torch.tensor([[-1, 0, 0, 2, 3]] * 2, dtype=torch.int32)
    choices = torch.tensor([[22, 0, 23, 9, 0], [7, 0, 0, 0, 0]])
    got = c.accept(tokens, parents, choices)
    assert got.lengths.tolist() == [3, 1] and got.next_tokens.tolist() == [9, 7]
    assert held(c, 1) == every(list(range(14)) + [20, 22, 23])
    assert held(c, 4) == every(list(range(100, 114)) + [120])
    assert c.seq_lens_tensor().tolist() == [17, 15]
    grow(c, [1, 4], [[30], [130]])
    assert held(c, 1) == every(list(range(14)) + [20, 22, 23, 30])


def test_accept_leaves_a_fork_alone_and_asks_for_all_active_sequences(plain):
    c = cache()
    grow(c, [0], [list(range(20))])
    c.fork(0, [2])
    grow(c, [0], [[50, 51, 52]])
    tokens = torch.tensor([[50, 51, 52]])
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    with pytest.raises(ValueError, match="tokens"):
        c.accept(tokens.repeat(2, 1), parents.repeat(2, 1), tokens.repeat(2, 1))
    with pytest.raises(ValueError, match="drafted"):
        c.accept(torch.zeros(1, 40, dtype=torch.long), parents, tokens)
    c.accept(tokens, parents, torch.tensor([[52, 0, 0]]))
    assert held(c, 0) == every(list(range(20)) + [50, 52])
    assert held(c, 2) == every(range(20))


def test_accept_bounds_the_pages_it_moved(plain):
    c = cache()
    c.kmin = [torch.full((c.num_blocks, H, D), 9e9) for _ in range(LAYERS)]
    c.kmax = [torch.full((c.num_blocks, H, D), -9e9) for _ in range(LAYERS)]
    kmin, kmax, c.kmin, c.kmax = c.kmin, c.kmax, None, None
    grow(c, [0], [list(range(14))])
    grow(c, [0], [list(range(40, 64))])
    c.kmin, c.kmax = kmin, kmax
    parents = torch.tensor([[-1] + list(range(23))], dtype=torch.int32)
    choices = torch.tensor([list(range(41, 61)) + [0] * 4])
    c.accept(torch.tensor([list(range(40, 64))]), parents, choices)
    t = c.tables[0]
    assert t.length == 35
    numbers = list(range(14)) + list(range(40, 61))
    for page in range(3):
        rows = numbers[16 * page:16 * page + 16]
        for li in range(LAYERS):
            assert (c.kmin[li][t.blocks[page]] == min(rows) + 1000 * li).all()
            assert (c.kmax[li][t.blocks[page]] == max(rows) + 1000 * li).all()


def sums_for(c, slot, wanted):
    """Sums of a slot with which the positions `wanted` [layer][head] are kept."""
    for li in range(LAYERS):
        for h in range(H):
            c.weight_sums[li, slot, h, :c.tables[slot].length] = 0.25
            c.weight_sums[li, slot, h, wanted[li][h]] = 2.0


def test_evict_keeps_a_budget_and_gives_pages_back(plain):
    c = cache()
    c.enable_weight_sums()
    grow(c, [0, 3, 5], [list(range(70)), list(range(100, 170)), list(range(200, 270))])
    c.rewind(30, slots=[5])
    wanted = [[[10, 40], [11, 69 - 9]], [[12, 13], [33, 14]]]
    sums_for(c, 0, wanted)
    sums_for(c, 3, wanted)
    used = c.allocator.num_used
    assert c.evict(33, sinks=3, recent=8) == [0, 3]
    assert used - c.allocator.num_used == 2 * 2                  # of five pages, three are left
    for slot, first in ((0, 0), (3, 100)):
        for li in range(LAYERS):
            for h in range(H):
                got = held(c, slot)[li][h]
                assert len(got) == 33 and got == sorted(got)
                assert got[:3] == [first, first + 1, first + 2]
                assert got[-8:] == [first + 62 + i for i in range(8)]
                assert {first + p for p in wanted[li][h]} <= set(got)
                s = c.weight_sums[li, slot, h]
                assert (s[33:] == 0).all() and (s[:33] > 0).all()
                assert [i for i in range(33) if s[i] == 2.0] == \
                    sorted(got.index(first + p) for p in wanted[li][h])
    assert c.tables[5].length == 30 and len(held(c, 5)[0][0]) == 30
    assert c.seq_lens_tensor().tolist() == [33, 33, 30]
    assert c.block_tables_tensor()[0, :3].tolist() == c.tables[0].blocks
    assert c.evict(33) == []
    assert c.seq_positions == [70, 70, 30]
    grow(c, [0, 3, 5], [[90], [190], [290]])                      # and the sequence goes on
    assert c.seq_positions == [71, 71, 31]
    assert held(c, 0)[1][0][-1] == 90


def test_evict_copies_pages_that_others_hold(plain):
    c = cache()
    prefix = PrefixCache(c.allocator, 16)
    c.enable_weight_sums()
    grow(c, [0], [list(range(64))])
    prefix.register(list(range(64)), c.tables[0].blocks[:c.shareable_blocks(0)])
    c.fork(0, [1])
    c.weight_sums[:, :2, :, 20:40] = 1.0
    assert c.evict(24, sinks=2, recent=2, slots=[0]) == [0]
    assert held(c, 1) == every(range(64))                        # the fork, and the prefix's pages
    assert held(c, 0) == every([0, 1] + list(range(20, 40)) + [62, 63])
    assert c.shareable_blocks(0) == 0 and c.shareable_blocks(1) == 4
    assert prefix.match(list(range(64)) + [7]) == c.tables[1].blocks
    c.fork(0, [2])
    assert c.shareable_blocks(2) == 0
    c.free_sequence(0)
    grow(c, [0], [list(range(16))])
    assert c.shareable_blocks(0) == 1
    assert (c.weight_sums[:, 0] == 0).all()                      # a new sequence's start


def test_evict_without_blocks_for_the_copies_changes_nothing(plain):
    c = cache(blocks=5)
    c.enable_weight_sums()
    grow(c, [0], [list(range(64))])
    c.fork(0, [1])
    grow(c, [1], [[99]])
    before = [list(t.blocks) for t in c.tables], c.weight_sums.clone()
    with pytest.raises(OutOfBlocks):
        c.evict(40, slots=[0])
    assert [list(t.blocks) for t in c.tables] == before[0]
    assert torch.equal(c.weight_sums, before[1]) and held(c, 0) == every(range(64))


def test_sums_follow_a_sequence(plain):
    c = cache()
    with pytest.raises(RuntimeError, match="enable_weight_sums"):
        c.evict(8)
    grow(c, [2, 0], [list(range(30)), list(range(30))])
    c.enable_weight_sums()
    assert c.sum_rows_tensor().tolist() == [2, 0]
    c.weight_sums[:] = 1.0
    c.rewind(12, slots=[2])
    assert (c.weight_sums[:, 2, :, 12:] == 0).all() and (c.weight_sums[:, 2, :, :12] == 1).all()
    c.fork(2, [4])
    assert torch.equal(c.weight_sums[:, 4], c.weight_sums[:, 2])
    for bad in (0, -3):
        with pytest.raises(ValueError, match="budget"):
            c.evict(bad)
    with pytest.raises(ValueError, match="does not hold"):
        c.evict(8, sinks=4, recent=5)


def test_selection_of_rows_longer_than_any_cache_is_refused():
    from latentserve_amd import _tree
    lib = _tree.lib()
    st = (ctypes.c_int64 * 3)(1 << 33, 1 << 33, 1 << 32)
    args = (st, (1 << 30) + 1, 64, 1 << 13, 1 << 14, 1, 1, 1, 8, 1, 1, None)
    assert lib.ls_select_tokens(1 << 12, *args) == 1


def test_a_pool_listed_twice_is_refused():
    a, b, c = (torch.zeros(4, 16, 2, 128, dtype=torch.float16) for _ in range(3))
    tables, lens = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    keep = torch.zeros(2, 1, 2, 3, dtype=torch.int32)
    one = torch.zeros(1, 1, dtype=torch.int64)
    for k, v in (([a, a], [b, c]), ([a, b], [c, a]), ([a, b], [a, b])):
        with pytest.raises(ValueError, match="twice"):
            ce.move_tokens(keep, k, v, tables, lens)
        with pytest.raises(ValueError, match="twice"):
            ta.accept_tokens(one, one.int(), one, k, v, tables, lens)


def test_a_bounded_sequence_ends_where_the_positions_do(plain):
    c = cache()
    c.max_positions = 70
    c.enable_weight_sums()
    grow(c, [0, 1], [list(range(60)), list(range(60))])
    c.evict(20, sinks=1, recent=4, slots=[0])
    grow(c, [0], [list(range(60, 70))])
    assert c.seq_positions == [70] and c.seq_lens == [30]
    c.fork(0, [2])
    for slots in ([0], [1, 2]):
        before = [list(t.blocks) for t in c.tables], [t.length for t in c.tables]
        with pytest.raises(RuntimeError, match="position 70"):
            c.advance(1, slots=slots)
        assert ([list(t.blocks) for t in c.tables], [t.length for t in c.tables]) == before
    c.rewind(25, slots=[0])
    grow(c, [0], [[65]])
    c.free_sequence(0)
    grow(c, [0], [list(range(80))])                               # (no bound but the capacity)
    assert c.seq_positions == [80]
