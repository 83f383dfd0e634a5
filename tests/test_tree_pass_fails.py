"""A pass over drafted trees that fails part way leaves nothing for accept() to go by: the
decoder on the CPU, with plain stand-ins for its layers and the attention."""

from __future__ import annotations

import pytest
import torch

from latentserve_amd.kernels.hip import cache_eviction as ce
from latentserve_amd.kernels.hip import tree_attention as ta
from latentserve_amd.runtime.qwen_decoder import DecoderConfig, QwenDecoder
from tests.test_bounded_cache import plain_accept

LAYERS = 3


@pytest.fixture
def decoder(monkeypatch):
    m = QwenDecoder(DecoderConfig(vocab_size=64, hidden_size=64, intermediate_size=32, num_layers=LAYERS,
                                  num_heads=2, num_kv_heads=1), device="cpu")
    m.allocate_cache(2, 64)
    m.cache.enable_weight_sums()
    m.added = []
    monkeypatch.setattr(ta, "accept_tokens", plain_accept)
    monkeypatch.setattr(ce, "add_weights", lambda q, lse, k, t, l, sums, **kw: m.added.append(len(m.added)))

    def layers(tokens, pos, slots, attend, bounds):
        q = torch.zeros(tokens.numel(), 1, 2, 128)
        for li in range(LAYERS):
            attend(li, m.layers[li], q, torch.empty_like(q), None, None)
        return torch.zeros(tokens.numel(), 64)

    m._run_layers = layers
    return m


def fails_in(monkeypatch, layer):
    calls = []

    def attention(*a, **kw):
        calls.append(0)
        if len(calls) - 1 == layer:
            raise RuntimeError("out of memory")

    monkeypatch.setattr(ta, "tree_attention", attention)


TOKENS = torch.tensor([[5, 6, 7], [8, 9, 10]])
PARENTS = torch.tensor([[-1, 0, 1]] * 2, dtype=torch.int32)
MASKS = torch.tensor([[[1], [3], [7]]] * 2)


def run(m):
    return m.tree_forward(TOKENS, TOKENS, MASKS, max_position=10)


@pytest.mark.parametrize("layer", range(LAYERS))
def test_a_failed_pass_is_not_accepted(decoder, monkeypatch, layer):
    m = decoder
    m.cache.advance(3)
    fails_in(monkeypatch, layer)
    with pytest.raises(RuntimeError, match="memory"):
        run(m)
    with pytest.raises(RuntimeError, match="tree_forward"):
        m.accept(TOKENS, PARENTS, TOKENS)
    assert m.added == [] and m.cache.seq_lens == [3, 3]
    fails_in(monkeypatch, None)                            # the pass made again
    run(m)
    m.accept(TOKENS, PARENTS, torch.tensor([[6, 0, 0], [9, 10, 0]]))
    assert len(m.added) == LAYERS and m.cache.seq_lens == [2, 3]


def test_nor_is_the_pass_before_it(decoder, monkeypatch):
    m = decoder
    m.cache.advance(3)
    fails_in(monkeypatch, None)
    run(m)
    fails_in(monkeypatch, 0)
    with pytest.raises(RuntimeError, match="memory"):
        run(m)
    with pytest.raises(RuntimeError, match="tree_forward"):
        m.accept(TOKENS, PARENTS, TOKENS)
    assert m.cache.seq_lens == [3, 3]
