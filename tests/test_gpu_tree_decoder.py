"""Drafted trees and a bounded cache through the decoder, on an MI355X: a tree's pass, the
path kept, the weight sums of decode steps and paths, eviction, and graphed steps between."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_runtime import make_model, reference_logits  # noqa: E402

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]

# (the fp16 pipeline against the fp32 forward: what the decode step is held to)
LOGITS, SMALL = 2e-2, 1e-3
# A row's weights add up to 1.  Scores of up to 40 whose 128 products are added in another
# order differ by at most 128 x 2^-24 x 40 = 3e-4, the exponential and the sum add less.
ONE = 1e-3


def tree(m, n=9, batch=2, seed=0):
    """A tree of each sequence, different ones, and choices that confirm a path of it."""
    g = torch.Generator().manual_seed(seed)
    parents = torch.full((batch, n), -1, dtype=torch.int32)
    tokens = torch.randint(0, m.cfg.vocab_size, (batch, n), generator=g)
    for b in range(batch):
        for i in range(1, n):
            parents[b, i] = int(torch.randint(0, i, (1,), generator=g))
        for i in range(n):                             # (siblings' tokens differ)
            tokens[b, i] = (tokens[b, i] // n) * n % m.cfg.vocab_size + i
    tokens %= m.cfg.vocab_size
    path = []
    choices = torch.full((batch, n), m.cfg.vocab_size + 5, dtype=torch.long)
    for b in range(batch):
        at, p = n - 1 - b, []
        while at >= 0:
            p.insert(0, at)
            at = int(parents[b, at])
        for x, y in zip(p, p[1:]):
            choices[b, x] = tokens[b, y]
        path.append(p)
    return tokens.cuda(), parents.cuda(), choices.cuda(), path


def context(m, steps, batch=2, seed=3):
    ids = torch.randint(0, m.cfg.vocab_size, (batch, steps),
                        generator=torch.Generator().manual_seed(seed)).cuda()
    for t in range(steps):
        m.cache.advance(1, batch_size=batch)
        pos = torch.full((batch, 1), t, dtype=torch.long, device="cuda")
        m.decode_forward_static(ids[:, t:t + 1], pos, max_position=t)
    return ids


def tree_pass(m, tokens, parents, start):
    from latentserve_amd.kernels.hip.tree_attention import tree_masks
    masks, depths = tree_masks(parents)
    m.cache.advance(tokens.shape[1], batch_size=tokens.shape[0])
    return m.tree_forward(tokens, start + depths.long(), masks, max_position=start + tokens.shape[1])


def close(got, want):
    err = (got.float() - want).abs().max().item()
    assert err <= LOGITS * want.abs().max().item() + SMALL, err


@pytest.mark.parametrize("steps,n", [(1, 9), (37, 9), (20, 50)])
def test_every_node_sees_its_path(steps, n):
    m = make_model(cap=128, batch=2, seed=2)
    ids = context(m, steps)
    tokens, parents, _, _ = tree(m, n)
    logits = tree_pass(m, tokens, parents, steps)
    for b in range(2):
        for i in range(tokens.shape[1]):
            at, p = i, []
            while at >= 0:
                p.insert(0, at)
                at = int(parents[b, at])
            close(logits[b, i], reference_logits(m, torch.cat([ids[b], tokens[b, p]])[None])[0])


def test_the_kept_path_is_the_context_of_the_next_step():
    m = make_model(cap=128, batch=2, seed=4)
    ids = context(m, 30)
    m.cache.enable_weight_sums()
    for turn in range(3):
        tokens, parents, choices, path = tree(m, n=5 + 6 * turn, seed=turn)
        lens = m.cache.seq_lens
        start = torch.tensor(lens, device="cuda")[:, None]
        from latentserve_amd.kernels.hip.tree_attention import tree_masks
        masks, depths = tree_masks(parents)
        n = tokens.shape[1]
        m.cache.advance(n, batch_size=2)
        m.tree_forward(tokens, start + depths.long(), masks, max_position=max(lens) + n)
        got = m.accept(tokens, parents, choices)
        assert got.lengths.tolist() == [len(p) for p in path]
        if turn == 0:
            ids = [ids[0], ids[1]]
        ids = [torch.cat([ids[b], tokens[b, path[b]]]) for b in range(2)]
        assert m.cache.seq_lens == [len(x) for x in ids]
    m.cache.advance(1, batch_size=2)
    nxt = torch.tensor([[7], [11]], device="cuda")
    pos = torch.tensor([[len(x)] for x in ids], device="cuda")
    logits = m.decode_forward_static(nxt, pos, max_position=int(pos.max()))
    for b in range(2):
        close(logits[b, 0], reference_logits(m, torch.cat([ids[b], nxt[b]])[None])[0])
    # every row of the accepted tokens and of the step gave its weights once
    rep = m.cfg.num_heads // m.cfg.num_kv_heads
    for b in range(2):
        sums = m.cache.weight_sums[:, b].double()
        length = m.cache.tables[b].length
        want = rep * (len(ids[b]) - 30 + 1)
        assert ((sums.sum(-1) - want).abs() <= ONE * want).all()
        assert (sums[..., length:] == 0).all() and (sums[..., :length] > 0).all()


@pytest.mark.parametrize("kv_dtype", ["int8", "int4"])
def test_quantized_caches_are_refused(kv_dtype):
    m = make_model(cap=64, batch=2, seed=4)
    m.allocate_cache(2, 64, kv_dtype=kv_dtype)
    tokens, parents, choices, _ = tree(m)
    with pytest.raises(ValueError, match="fp16"):
        m.tree_forward(tokens, tokens, parents, max_position=20)
    with pytest.raises(ValueError, match="fp16"):
        m.accept(tokens, parents, choices)


def test_accept_without_its_pass_is_refused():
    m = make_model(cap=64, batch=2, seed=4)
    m.cache.enable_weight_sums()
    context(m, 9)
    tokens, parents, choices, _ = tree(m)
    with pytest.raises(RuntimeError, match="tree_forward"):
        m.accept(tokens, parents, choices)
    m.cache.advance(9, batch_size=2)
    m.sparse_ratio = 0.5
    with pytest.raises(ValueError, match="sparse"):
        m.decode_forward_static(tokens[:, :1], tokens[:, :1], max_position=20)


def test_a_trees_pages_have_their_bounds():
    m = make_model(cap=128, batch=2, seed=5)
    m.set_sparse(0.5)
    m.set_sparse(None)
    context(m, 14)
    m.cache.enable_page_bounds()
    tokens, parents, choices, _ = tree(m, n=23)
    tree_pass(m, tokens, parents, 14)
    m.accept(tokens, parents, choices)
    c = m.cache
    for b in range(2):
        t = c.tables[b]
        for li, pool in enumerate(c.k_pool):
            for page, blk in enumerate(t.blocks[:-(-t.length // 16)]):
                if page == 0 and t.length >= 16 or page > 0:
                    live = pool[blk, :min(16, t.length - 16 * page)]
                    assert torch.equal(c.kmin[li][blk], live.amin(0))
                    assert torch.equal(c.kmax[li][blk], live.amax(0))


@pytest.mark.parametrize("graphed", [False, True])
def test_a_bounded_cache_keeps_what_got_attention(graphed):
    from latentserve_amd.runtime.hip_graph import GraphedDecoder

    m = make_model(cap=96, batch=3, seed=6)
    m.allocate_cache(3, 96, max_positions=256)
    m.cache.enable_weight_sums()
    dec = GraphedDecoder(m, buckets=(32, 64), enabled=graphed)
    ids = torch.randint(0, m.cfg.vocab_size, (3, 150), generator=torch.Generator().manual_seed(1)).cuda()
    rep = m.cfg.num_heads // m.cfg.num_kv_heads
    c, steps = m.cache, 0
    for t in range(150):
        pos = torch.full((3, 1), t, dtype=torch.long, device="cuda")
        out = dec.step(ids[:, t:t + 1], pos, slots=[2, 0, 1])
        steps += 1
        assert c.seq_positions == [t + 1] * 3
        assert out.isfinite().all()
        if c.max_len < 90:
            continue
        # each row's weights once, warm-ups and recordings aside
        want = rep * steps
        total = c.weight_sums.double().sum(-1)
        assert ((total - want).abs() <= ONE * want).all()
        sums = c.weight_sums[..., :90].clone()
        rows = [[p.view(-1, 2, 128)[[c.tables[s].slot(i) for i in range(90)]].clone() for s in range(3)]
                for p in c.k_pool + c.v_pool]
        assert c.evict(48, sinks=4, recent=8) == [2, 0, 1]
        for s in range(3):
            for li in range(2):
                for h in range(2):
                    rank = sums[li, s, h].clone()
                    rank[:4] = rank[82:] = float("inf")
                    keep = rank.argsort(descending=True, stable=True)[:48].sort()[0]
                    assert torch.equal(c.weight_sums[li, s, h, :48], sums[li, s, h, keep])
                    for z, pool in ((li, c.k_pool[li]), (2 + li, c.v_pool[li])):
                        at = [c.tables[s].slot(i) for i in range(48)]
                        assert torch.equal(pool.view(-1, 2, 128)[at, h], rows[z][s][keep, h])
        assert (c.weight_sums[..., 48:] == 0).all()
        c.weight_sums.zero_()
        steps = 0
    assert c.max_len < 96 and t == 149
