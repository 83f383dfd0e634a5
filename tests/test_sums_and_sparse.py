"""Weight sums and sparse steps are refused together where they are put together, and by a
runner's step before the cache has advanced."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from latentserve_amd.runtime.hip_graph import GraphedDecoder
from latentserve_amd.runtime.qwen_decoder import DecoderConfig, QwenDecoder


def model():
    m = QwenDecoder(DecoderConfig(vocab_size=64, hidden_size=64, intermediate_size=32, num_layers=2,
                                  num_heads=2, num_kv_heads=1), device="cpu")
    m.allocate_cache(3, 64)
    m.cache.enable_page_bounds = lambda: setattr(m.cache, "bounded", True)
    return m


def test_sparse_steps_of_a_cache_that_sums_are_refused_when_set():
    m = model()
    m.cache.enable_weight_sums()
    with pytest.raises(ValueError, match="weights"):
        m.set_sparse(0.5, recent=7)
    assert m.sparse_ratio is None and not hasattr(m.cache, "bounded")
    assert m.layers[0].attn.sparse_recent == 2
    m.set_sparse(None)


def test_sums_beside_sparse_steps_are_refused_when_enabled():
    m = model()
    m.set_sparse(0.5)
    with pytest.raises(ValueError, match="weights"):
        m.cache.enable_weight_sums()
    assert m.cache.weight_sums is None
    m.allocate_cache(3, 64)                                # (the model's steps are sparse still)
    with pytest.raises(ValueError, match="weights"):
        m.cache.enable_weight_sums()
    m.cache.enable_page_bounds = lambda: None
    m.set_sparse(None)
    m.cache.enable_weight_sums()
    assert m.cache.weight_sums is not None


@pytest.mark.parametrize("by_policy", [False, True])
def test_a_refused_step_leaves_the_cache_as_it_was(by_policy):
    m = model()
    asked = []
    policy = SimpleNamespace(choose=lambda n, mean: asked.append((n, mean)) or 0.25) if by_policy else None
    dec = GraphedDecoder(m, enabled=False, policy=policy)
    m.cache.advance(5, slots=[0, 2])
    m.cache.enable_weight_sums()
    if not by_policy:
        m.sparse_ratio = 0.5
    ids = torch.zeros(2, 1, dtype=torch.long)
    for _ in range(3):
        with pytest.raises(ValueError, match="weights"):
            dec.step(ids, ids + 5, slots=[0, 2])
    assert [t.length for t in m.cache.tables] == [5, 0, 5]
    assert m.cache.seq_lens_tensor().tolist() == [5, 5]
    assert dec.stats()["ratio_tokens"] == {} and dec.eager_steps == 0
    assert asked == ([(2, 6.0)] * 3 if by_policy else [])  # (of the lengths that the step would have)
