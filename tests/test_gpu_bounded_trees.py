"""Drafted trees of sequences that lost tokens, on an MI355X: nodes at the positions that
follow all tokens there were, over the rows that were kept."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_runtime import make_model  # noqa: E402
from test_gpu_tree_decoder import ONE, close, context, tree  # noqa: E402

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def held_rows(c, slot):
    """K and V of a slot's tokens, [layers] of fp32 [H, length, D] each."""
    t = c.tables[slot]
    at = [t.slot(i) for i in range(t.length)]
    return [[p.flatten(0, 1)[at].float().transpose(0, 1) for p in pools] for pools in (c.k_pool, c.v_pool)]


def logits_behind(m, rows, tokens, start):
    """fp32 logits of the last of `tokens`, at positions from start on, behind cached rows."""
    cfg, n = m.cfg, len(tokens)
    hd, half, rep = cfg.head_dim, cfg.head_dim // 2, cfg.num_heads // cfg.num_kv_heads
    qd, kvd = cfg.num_heads * hd, cfg.num_kv_heads * hd
    pos = torch.arange(start, start + n, device="cuda")
    cos, sin = m.rope.cos[pos].float(), m.rope.sin[pos].float()

    def rope(z):                                           # [H, n, D]
        return z * cos + torch.cat([-z[..., half:], z[..., :half]], dim=-1) * sin

    def norm(z, w):
        return z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps) * w.float()

    x = m.embed[tokens].float()
    for li, layer in enumerate(m.layers):
        qkv = norm(x, layer.norm1) @ layer.w_qkv.float().T + layer.b_qkv.float()
        q = rope(qkv[:, :qd].view(n, cfg.num_heads, hd).transpose(0, 1))
        k = rope(qkv[:, qd:qd + kvd].view(n, cfg.num_kv_heads, hd).transpose(0, 1))
        v = qkv[:, qd + kvd:].view(n, cfg.num_kv_heads, hd).transpose(0, 1)
        k = torch.cat([rows[0][li], k], 1).repeat_interleave(rep, 0)
        v = torch.cat([rows[1][li], v], 1).repeat_interleave(rep, 0)
        s = q @ k.transpose(-1, -2).contiguous() / math.sqrt(hd)
        s = s + torch.full((n, k.shape[1]), float("-inf"), device="cuda").triu(k.shape[1] - n + 1)
        x = x + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, qd) @ layer.w_o.float().T
        g, u = (norm(x, layer.norm2) @ layer.w_gate_up.float().T).chunk(2, dim=-1)
        x = x + (torch.nn.functional.silu(g) * u) @ layer.w_down.float().T
    return norm(x[-1], m.norm) @ m.lm_head.float().T


def test_a_tree_behind_an_eviction():
    from latentserve_amd.kernels.hip.tree_attention import tree_masks

    m = make_model(cap=96, batch=2, seed=8)
    m.allocate_cache(2, 96, max_positions=256)
    c = m.cache
    c.enable_weight_sums()
    context(m, 70)
    assert c.evict(40, sinks=2, recent=9) == [0, 1]
    rep = m.cfg.num_heads // m.cfg.num_kv_heads
    for turn in range(3):                                  # (the second one's context: 40 rows and a path)
        starts = c.seq_positions
        assert all(p > n for p, n in zip(starts, c.seq_lens))
        rows = [held_rows(c, s) for s in range(2)]
        before, lens = c.weight_sums.double().sum(-1), c.seq_lens
        tokens, parents, choices, path = tree(m, n=7 + 8 * turn, seed=20 + turn)
        masks, depths = tree_masks(parents)
        c.advance(tokens.shape[1], batch_size=2)
        at = torch.tensor(starts, device="cuda")[:, None]
        print(f"tree of {tokens.shape[1]} behind {lens} rows at {starts}", flush=True)
        logits = m.tree_forward(tokens, at + depths.long(), masks, max_position=max(starts) + tokens.shape[1])
        for b in range(2):
            for i in range(tokens.shape[1]):
                node, p = i, []
                while node >= 0:
                    p.insert(0, node)
                    node = int(parents[b, node])
                close(logits[b, i], logits_behind(m, rows[b], tokens[b, p], starts[b]))
        got = m.accept(tokens, parents, choices)
        assert got.lengths.tolist() == [len(p) for p in path]
        assert c.seq_positions == [s + len(p) for s, p in zip(starts, path)]
        assert c.seq_lens == [n + len(p) for n, p in zip(lens, path)]
        # (each row of the path gave a weight of one, the path's tokens had none before)
        for b in range(2):
            gave = c.weight_sums.double().sum(-1)[:, b] - before[:, b]
            want = rep * len(path[b])
            assert ((gave - want).abs() <= ONE * (want + before[:, b])).all()
        if turn == 1:
            assert c.evict(36, sinks=2, recent=9) == [0, 1]
    # a decode step goes on from there
    starts, rows = c.seq_positions, [held_rows(c, s) for s in range(2)]
    nxt = torch.tensor([[7], [11]], device="cuda")
    c.advance(1, batch_size=2)
    logits = m.decode_forward_static(nxt, torch.tensor(starts, device="cuda")[:, None],
                                     max_position=max(starts))
    for b in range(2):
        close(logits[b, 0], logits_behind(m, rows[b], nxt[b], starts[b]))


def test_a_rewound_sequence_starts_anew():
    """After rewind(0) of an evicted sequence, the same tokens give the same logits as in a slot
    that never held any."""
    m = make_model(cap=96, batch=2, seed=9)
    m.allocate_cache(2, 96, max_positions=128)
    c = m.cache
    c.enable_weight_sums()
    context(m, 60)
    c.evict(30, sinks=2, recent=9)
    c.rewind(0, slots=[0])
    c.free_sequence(1)
    ids = torch.randint(0, m.cfg.vocab_size, (1, 80), generator=torch.Generator().manual_seed(2)).cuda()
    for t in range(80):
        c.advance(1, slots=[0, 1])
        pos = torch.tensor(c.seq_positions, device="cuda")[:, None] - 1
        assert pos.tolist() == [[t], [t]]
        logits = m.decode_forward_static(ids[:, t:t + 1].expand(2, 1).contiguous(), pos, max_position=t)
    assert torch.equal(logits[0], logits[1])
    assert torch.equal(c.weight_sums[:, 0], c.weight_sums[:, 1])
