"""Branching generation on an MI355X as a program uses it: a decoder over each paged
cache, a prompt forked into branches, decoded through captured graphs, ranked by log
probability, compacted, and decoded on."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]

KINDS = {"fp16": dict(), "int8": dict(kv_dtype="int8"), "int8 asym": dict(kv_dtype="int8", asymmetric=True),
         "int4": dict(kv_dtype="int4")}


def make(kind, batch=6, cap=192, blocks=None, seed=0):
    from latentserve_amd.runtime.qwen_decoder import DecoderConfig, QwenDecoder
    m = QwenDecoder(DecoderConfig(vocab_size=512, intermediate_size=384, num_layers=2), seed=seed,
                    std=0.05)
    m.allocate_cache(batch, cap, num_blocks=blocks, **KINDS[kind])
    return m


def step(m, slots, ids):
    """One eager decode step; logits [B, V]."""
    m.cache.advance(1, slots=slots)
    pos = torch.tensor([[m.cache.tables[s].length - 1] for s in slots], device="cuda")
    return m.decode_forward_static(ids.view(-1, 1), pos, max_position=m.cache.max_len)[:, 0]


def prompt_ids(n, seed=1):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 15, 16, 37, 48])
def test_a_branch_decodes_as_a_sequence_of_its_own(kind, length):
    """Forked at `length` tokens and grown apart: every branch's logits are those of the
    same tokens decoded from scratch (the same launches over the same entries; the
    order of a merge's sums may differ: 3e-3 of the largest, as the eager and graphed
    steps of the other tests)."""
    ids = prompt_ids(length)
    m = make(kind)
    for t in range(length):
        step(m, [0], ids[t])
    m.cache.fork(0, [1, 2])
    tails = torch.stack([prompt_ids(20, 10 + i) for i in range(3)])
    got = [step(m, [0, 1, 2], tails[:, t]) for t in range(20)]
    alone = make(kind)
    for t in range(length):
        step(alone, [3, 4, 5], ids[t].expand(3))
    for t in range(20):
        want = step(alone, [3, 4, 5], tails[:, t]).float()
        assert (got[t].float() - want).abs().max() <= 3e-3 * want.abs().max() + 1e-4, t


@pytest.mark.parametrize("kind", KINDS)
def test_compaction_changes_no_step(kind):
    ids = torch.stack([prompt_ids(45, 20 + i) for i in range(4)])
    runs = []
    for compact in (False, True):
        m = make(kind, blocks=40)
        for t in range(45):
            step(m, [0, 1, 2, 3], ids[:, t])
        m.cache.fork(2, [4])
        m.cache.free_sequence(0)
        m.cache.free_sequence(1)
        if compact:
            used = m.cache.allocator.num_used
            moves = m.cache.compact()
            assert moves and max(max(t.blocks, default=0) for t in m.cache.tables) < used
        runs.append([step(m, [2, 3, 4], prompt_ids(3, 30 + t)).float() for t in range(10)])
    for a, b in zip(*runs):
        assert (a - b).abs().max() <= 3e-3 * a.abs().max() + 1e-4


def test_int4_steps_follow_the_fp16_ones():
    """The 4-bit decoder against a reference that holds the same entries: an fp16 cache
    filled with what the 4-bit cache reads back gives the same attention."""
    from latentserve_amd.kernels.hip import int4_cache as i4
    from latentserve_amd.kernels.hip import paged_decode_hip as pdh
    m = make("int4", batch=3)
    ids = torch.stack([prompt_ids(60, 40 + i) for i in range(3)])
    for t in range(60):
        logits = step(m, [0, 1, 2], ids[:, t])
    assert torch.isfinite(logits).all()
    c = m.cache
    for li in range(2):
        k, v = c.read(li, 3)
        kp = torch.zeros(3 * 4, 16, 2, 128, dtype=torch.float16, device="cuda")
        vp = torch.zeros_like(kp)
        kp.view(3, 64, 2, 128)[:, :60] = k.transpose(1, 2)
        vp.view(3, 64, 2, 128)[:, :60] = v.transpose(1, 2)
        tab = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4)
        q = torch.randn(3, 2, 6, 128, generator=torch.Generator("cuda").manual_seed(li),
                        device="cuda").half()
        want = pdh.paged_decode_hip(q, kp, vp, tab, c.seq_lens_tensor(3), 64).float()
        got = i4.paged_decode_int4(q, c.pools[li], c.block_tables_tensor(3), c.seq_lens_tensor(3)).float()
        # two roundings of the weights and of the results, 2^-11 each of at most max |v|
        assert (got - want).abs().max() <= 4 * 2.0 ** -11 * v.abs().max().item()


def test_int4_prefill_in_chunks_is_the_tokens_one_by_one():
    from latentserve_amd.runtime.int4_cache import Int4PagedKVCache
    from latentserve_amd.runtime.kv_cache import KVCacheSpec
    spec = KVCacheSpec(num_layers=1, num_kv_heads=2, head_dim=128, max_batch_size=2, max_seq_len=128)
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(2, 2, 75, 128, generator=g, device="cuda").half() for _ in range(2))
    got = []
    for sizes in ([75], [30, 1, 44], [1] * 75):
        c, at = Int4PagedKVCache(spec), 0
        for n in sizes:
            c.advance(n, batch_size=2)
            c.write(0, k[:, :, at:at + n], v[:, :, at:at + n])
            at += n
        got.append(c.read(0, 2, 80))
        assert (got[-1][0][:, :, 75:] == 0).all()
    for a in got[1:]:
        assert torch.equal(a[0], got[0][0]) and torch.equal(a[1], got[0][1])
    c.rewind(20)
    c.advance(3)
    c.write(0, k[:, :, 70:73], v[:, :, 70:73])
    back = c.read(0, 2, 23)
    assert torch.equal(back[0][:, :, :20], got[0][0][:, :, :20])
    assert torch.equal(back[1][:, :, 20:], got[0][1][:, :, 70:73])


@pytest.mark.parametrize("kind", KINDS)
def test_graphed_branches_with_logprobs(kind):
    """The whole path: prompt, fork, graphed greedy steps with log probabilities, the
    best branch kept, the others freed, compaction, more graphed steps, beside an
    eager run of the same."""
    from latentserve_amd.runtime.hip_graph import GraphedDecoder
    runs = []
    for enabled in (True, False):
        m = make(kind, blocks=60)
        ids = prompt_ids(40)
        for t in range(40):
            step(m, [0], ids[t])
        m.cache.fork(0, [1, 2, 3])
        dec = GraphedDecoder(m, buckets=(64, 128), enabled=enabled, greedy=True, logprobs=4)
        tok = torch.tensor([[5], [6], [7], [8]], device="cuda")
        seen, total = [], torch.zeros(4, device="cuda")
        slots = [0, 1, 2, 3]
        for t in range(30):                              # crosses a bucket
            pos = torch.tensor([[m.cache.tables[s].length] for s in slots], device="cuda")
            nxt = dec.step_greedy(tok, pos, slots).clone()
            s = dec.last_logprobs
            assert torch.equal(s.top_ids[:, :1], nxt) and torch.equal(s.top_logprobs[:, 0], s.logprob)
            assert (s.entropy > 0).all() and (s.top_logprobs[:, :3] >= s.top_logprobs[:, 1:]).all()
            total = total + s.logprob
            tok = nxt
            seen.append(s.logprob.clone())
            if t == 14:
                best = int(total.argmax())
                for x in slots:
                    if x != best:
                        m.cache.free_sequence(x)
                m.cache.compact()
                kids = [x for x in slots if x != best][:2]
                m.cache.fork(best, kids)
                slots = [best] + kids
                tok = torch.stack([tok[best], tok[best] + 1, tok[best] + 2]) % 512
                total = torch.zeros(3, device="cuda")
        runs.append(seen)
        if enabled:
            assert dec.stats()["graph_steps"] == 30 and dec.stats()["captures"] >= 2
    # the first step's inputs are the same in both runs (later ones may part where two
    # logits nearly tie)
    a, b = runs[0][0], runs[1][0]
    assert (a - b).abs().max() <= 2e-2
    assert np.isfinite([x.cpu().numpy().sum() for x in runs[0]]).all()


def test_logprobs_need_greedy_and_sparse_needs_fp16():
    from latentserve_amd.runtime.hip_graph import GraphedDecoder
    m = make("int4")
    with pytest.raises(ValueError):
        GraphedDecoder(m, logprobs=3)
    with pytest.raises(ValueError):
        m.set_sparse(0.5)
    with pytest.raises(ValueError):
        m.allocate_cache(2, 64, kv_dtype="int2")


def test_fork_and_rewind_keep_the_page_bounds_of_sparse_decode():
    """Branches of an fp16 cache with page bounds: after a fork, a rewind and growth, the
    bounds of every held page are its keys' minimum and maximum or wider, and
    those of the untouched branch unchanged."""
    from latentserve_amd.runtime.kv_cache import KVCacheSpec, PagedKVCache
    spec = KVCacheSpec(num_layers=2, num_kv_heads=2, head_dim=128, max_batch_size=3, max_seq_len=128)
    c = PagedKVCache(spec)
    c.enable_page_bounds()
    g = torch.Generator("cuda").manual_seed(5)

    def write(n, slots):
        c.advance(n, slots=slots)
        for li in range(2):
            x = torch.randn(len(slots), 2, n, 128, generator=g, device="cuda").half()
            c.write(li, x, x)

    write(40, [0])
    c.fork(0, [1])
    kept = [c.kmin[li][c.tables[0].blocks[:3]].clone() for li in range(2)]
    c.rewind(35, slots=[1])
    write(1, [1])
    for li in range(2):
        assert torch.equal(c.kmin[li][c.tables[0].blocks[:3]], kept[li])
        for s in (0, 1):
            t = c.tables[s]
            for p, blk in enumerate(t.blocks):
                rows = c.k_pool[li][blk][:min(16, t.length - 16 * p)]
                if len(rows):
                    assert (c.kmin[li][blk] <= rows.amin(0)).all()
                    assert (c.kmax[li][blk] >= rows.amax(0)).all()
    assert c.tables[0].blocks[2] != c.tables[1].blocks[2]
