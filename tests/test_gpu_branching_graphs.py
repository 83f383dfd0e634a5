"""Captured decode steps of branches against eager steps of the same tokens, every step, on
an MI355X: forks, pages copied before they are written, a bucket crossed, compactions
under graphs that were recorded before them, freed and forked slots."""

from __future__ import annotations

import pytest

from tests.test_gpu_branching import KINDS, make, prompt_ids, step

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]

STEPS, TOP = 34, 4


def decode(m, advance, compact):
    """One program: an older sequence, a prompt and its branches, each step's tokens given.
    `advance(slots, ids)` makes a step and returns its logits [B, V]; yields them."""
    older, ids = prompt_ids(33, 50), prompt_ids(37, 51)
    for t in older:
        step(m, [4], t)
    for t in ids:
        step(m, [0], t)
    m.cache.fork(0, [1, 2, 3])
    slots = [0, 1, 2, 3]
    feed = torch.stack([prompt_ids(STEPS, 60 + i) for i in range(4)]).cuda()
    for t in range(STEPS):
        if t == 8:
            m.cache.free_sequence(4)                  # the pool's first blocks
            assert not compact or m.cache.compact()
        if t == 15:                                   # slot 2's branch, forked again
            for s in (0, 1, 3):
                m.cache.free_sequence(s)
            assert not compact or m.cache.compact() is not None
            m.cache.fork(2, [0, 1, 3])
        if t == 23:
            m.cache.free_sequence(1)                  # one ends, another takes its slot
            m.cache.fork(3, [1])
        yield advance(slots, feed[:, t])


@pytest.mark.parametrize("kind", KINDS)
def test_every_graphed_step_is_the_eager_one(kind):
    """The sums of a split launch have another order than an eager call's: 3e-3 of the
    largest logit, as between batches; in 8 and 4 bits a code that such a rounding tips moves
    its entry by a step: 2e-2.  Two branches lie further apart than that."""
    from latentserve_amd.runtime.hip_graph import GraphedDecoder
    graphed, eager = make(kind, blocks=60), make(kind, blocks=60)
    dec = GraphedDecoder(graphed, buckets=(64, 128), greedy=True, logprobs=TOP)
    chosen = []

    def by_graph(slots, ids):
        pos = torch.tensor([[graphed.cache.tables[s].length] for s in slots], device="cuda")
        chosen.append(dec.step_greedy(ids.view(-1, 1), pos, slots).clone())
        logits = dec._last_graph.logits_buf[:, 0].clone()
        check_scores(dec.last_logprobs, chosen[-1], logits)
        return logits

    apart = 0.0
    rel = 3e-3 if kind == "fp16" else 2e-2
    runs = zip(decode(graphed, by_graph, True), decode(eager, lambda s, i: step(eager, s, i), False))
    for t, (got, want) in enumerate(runs):
        got, want = got.float(), want.float()
        tol = rel * want.abs().max() + 1e-4
        off = (got - want).abs().max()
        assert off <= tol, (t, off.item(), tol.item())
        apart = max(apart, ((want[0] - want[1]).abs().max() / tol).item())
    assert apart > 5
    assert dec.stats()["graph_steps"] == STEPS and dec.stats()["captures"] == 2
    for p, q in zip(graphed.cache.tables[:4], eager.cache.tables[:4]):
        assert p.length == q.length and len(p.blocks) == len(q.blocks)


def check_scores(scores, nxt, logits):
    """Of these logits, in 64 bits (the bounds of tests/test_gpu_logprobs.py)."""
    logp = torch.log_softmax(logits.double(), -1)
    ids = torch.sort(logits.double(), dim=-1, descending=True, stable=True)[1][:, :TOP]
    assert torch.equal(scores.top_ids, ids) and torch.equal(nxt[:, 0], ids[:, 0])
    want = logp.gather(1, ids)
    near = lambda a, b: ((a.double() - b).abs() <= 2.0 ** -16 + 2.0 ** -16 * b.abs()).all()  # noqa: E731
    assert near(scores.top_logprobs, want) and near(scores.logprob, want[:, 0])
    assert near(scores.entropy, -(logp.exp() * logp).sum(-1))
