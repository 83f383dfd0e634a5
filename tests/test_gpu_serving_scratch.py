"""Scratch of captured and of large calls on an MI355X: a graph's counters serve later graphs
once it is gone, a large call's records are not kept."""

from __future__ import annotations

import gc

import pytest

from tests.test_gpu_branching import make, prompt_ids, step
from tests.test_gpu_int4_cache import attend_case, check, dev, i4, pools_of
from tests.test_gpu_logprobs_forms import check as check_scores

torch = pytest.importorskip("torch")

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.fixture
def small_slabs(monkeypatch):
    from latentserve_amd import _serving
    torch.cuda.synchronize()
    for name, value in (("_slabs", {}), ("_kept", []), ("_free", {}), ("_SLAB_INTS", 1 << 14)):
        monkeypatch.setattr(_serving, name, value, raising=name != "_free")
    return _serving


def test_decoders_made_again_and_again_take_no_more_counters(small_slabs):
    """Each captures a step of 8 sequences for 4096 tokens, 2048 counters a layer."""
    from latentserve_amd.runtime.hip_graph import GraphedDecoder
    m, alone = (make("int4", batch=8, cap=4096, blocks=400) for _ in range(2))
    ids = torch.stack([prompt_ids(40, i) for i in range(8)])
    slots = list(range(8))
    tok = [x.view(8, 1) for x in ids.t().contiguous()]
    for t in range(40):
        dec = GraphedDecoder(m, buckets=(), greedy=True, logprobs=2)
        pos = torch.tensor([[m.cache.tables[s].length] for s in slots], device="cuda")
        dec.step_greedy(tok[t], pos, slots)
        got = dec._last_graph.logits_buf[:, 0].float()
        want = step(alone, slots, tok[t]).float()
        # (in 4 bits a code that a rounding tips moves its entry by a step)
        assert (got - want).abs().max() <= 2e-2 * want.abs().max(), t
        del dec, got
        gc.collect()
    assert len(small_slabs._kept) <= 2, len(small_slabs._kept)


def test_graphs_after_others_and_beside_one_that_lives(small_slabs):
    q, arrays, tables, ln = attend_case([3000, 500, 40], seed=80)
    args = (dev(q), pools_of(arrays), dev(tables), dev(ln))
    i4().paged_decode_int4(*args)

    def record():
        g = torch.cuda.CUDAGraph()
        with small_slabs.counters_of(g), torch.cuda.graph(g):
            outs = [i4().paged_decode_int4(*args) for _ in range(2)]
        return g, outs

    kept, kept_outs = record()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(12):
        g, outs = record()
        for _ in range(3):
            for o in outs + kept_outs:
                o.zero_()
            torch.cuda.synchronize()
            for s, x in zip(streams, (kept, g)):
                with torch.cuda.stream(s):
                    x.replay()
            i4().paged_decode_int4(*args)
            torch.cuda.synchronize()
            for o in outs + kept_outs:
                check(o, q, arrays, tables, ln, rep)
        del g
        gc.collect()
    assert len(small_slabs._kept) <= 2


def test_the_records_of_a_large_call_are_not_kept():
    from latentserve_amd import _serving
    rows, n = 32768, 16378                               # two parts a row, 17.8 MB of records
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.empty(rows, n, dtype=torch.float16, device="cuda").normal_(generator=g)
    tok = torch.randint(0, n, (rows,), generator=g, device="cuda")
    from latentserve_amd.kernels.logprobs import token_logprobs
    out = token_logprobs(x, tok, 32)
    torch.cuda.synchronize()
    key = (0, torch.cuda.current_stream().cuda_stream)
    assert _serving._by_stream[key][0].numel() <= 16 << 20 if key in _serving._by_stream else True
    part = torch.arange(0, rows, 997, device="cuda")
    small = check_scores(x[part], tok[part], 32, 64)
    for a, b in zip(out, small):
        assert torch.equal(a[part], b)
