"""GraphedDecoder refuses a number of alternatives that its steps could not give, when it is
made: a step that fails has advanced the cache."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from latentserve_amd.runtime.hip_graph import GraphedDecoder


def model(vocab):
    return SimpleNamespace(device=torch.device("cpu"), rope=None,
                           cache=SimpleNamespace(spec=SimpleNamespace(max_seq_len=64)),
                           cfg=SimpleNamespace(vocab_size=vocab))


@pytest.mark.parametrize("vocab,good,bad", [(1000, (0, 1, 32), (-1, 33, 1000)), (20, (0, 20), (21, 32))])
def test_alternatives(vocab, good, bad):
    for k in good:
        assert GraphedDecoder(model(vocab), greedy=True, logprobs=k).logprobs == k
    for k in bad:
        with pytest.raises(ValueError, match="logprobs must be in"):
            GraphedDecoder(model(vocab), greedy=True, logprobs=k)
    assert GraphedDecoder(model(vocab), greedy=True).logprobs is None
