"""Log probabilities of given tokens on a HIP kernel, with each row's entropy and most
likely alternatives: what ranks the branches of a prompt, scores a prompt's own
tokens, and what a sampler reports beside its choice.

One launch that reads the logits once; beside it stand fused_elementwise's
argmax_rows (the greedy choice) and the decode step that makes the logits.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from latentserve_amd import _lib, _serving

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                   # [...] fp32
    entropy: torch.Tensor                   # [...] fp32, in nats
    top_logprobs: Optional[torch.Tensor]    # [..., top] fp32, largest first
    top_ids: Optional[torch.Tensor]         # [..., top] int64


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits [..., n] fp16 or fp32, tokens [...] int64 -> log softmax(logits)[tokens],
    the entropy of softmax(logits), and with top (0..32) the largest log
    probabilities and their tokens (equal logits: the lower number first).

    A token outside [0, n) is padding and gets 0.  Logits of -inf have probability
    0 (their log probability is -inf); a row of nothing else has entropy 0.  A NaN
    or +inf makes its row NaN (NaN ranks first).  No gradient is recorded."""
    if logits.dtype not in (torch.float16, torch.float32):
        raise ValueError(f"logits must be float16 or float32, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., n]")
    lead, n = logits.shape[:-1], logits.shape[-1]
    flat = len(lead) == 1
    if tokens.dtype != torch.int64 or tokens.shape != lead:
        raise ValueError(f"tokens must be int64 {tuple(lead)}, got {tokens.dtype} "
                         f"{tuple(tokens.shape)}")
    dev = logits.device
    if tokens.get_device() != logits.get_device():
        raise ValueError("tokens must be on the logits' device")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("logits require a gradient, which token_logprobs does not record")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, n):
        raise ValueError(f"top must be in [0, {min(MAX_TOP, n)}], got {top}")
    stream = _lib.stream_of(dev)
    if dev.index != _serving.current_device():
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top)
    x = logits if flat else logits.reshape(-1, n)
    if n > 1 and x.stride(1) != 1:
        x = x.contiguous()
    tok = tokens if flat else tokens.reshape(-1)
    rows = x.shape[0]
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    val = ids = None
    if top:
        val = torch.empty(rows, top, dtype=torch.float32, device=dev)
        ids = torch.empty(rows, top, dtype=torch.int64, device=dev)
    if rows:
        need, ints = _sizes(rows, n, top)
        work = cnt = None
        if need:
            work, cnt = _serving.scratch(dev, stream, need, ints)
        rc = _serving.lib().ls_token_logprobs(
            x.data_ptr(), x.stride(0) if rows > 1 else n, x.element_size(), tok.data_ptr(),
            tok.stride(0) if rows > 1 else 1, logprob.data_ptr(), entropy.data_ptr(),
            _lib.ptr(val), _lib.ptr(ids), _lib.ptr(work), need, _lib.ptr(cnt), rows, n, top, stream)
        _lib.check(rc, "ls_token_logprobs")
    if flat:
        return TokenLogprobs(logprob, entropy, val, ids)
    return TokenLogprobs(logprob.view(lead), entropy.view(lead),
                         None if val is None else val.view(*lead, top),
                         None if ids is None else ids.view(*lead, top))


# Workspace bytes and counters by a call's sizes.
_SIZES: dict = {}


def _sizes(rows: int, n: int, top: int):
    got = _SIZES.get((rows, n, top))
    if got is None:
        if max(rows, n) >= 1 << 31:                       # (C ints)
            raise ValueError(f"{rows} rows of {n} logits are too many for one call")
        lib = _serving.lib()
        got = (lib.ls_token_logprobs_workspace_bytes(rows, n, top),
               lib.ls_token_logprobs_counter_ints(rows, n, top))
        if len(_SIZES) >= 4096:
            _SIZES.clear()
        _SIZES[rows, n, top] = got
    return got
