"""ctypes binding of the second header, include/latentserve_amd_serving.h: the 4-bit
paged cache, page copies and token log probabilities.

The entry points live in the same liblatentserve_hip.so as ``_lib``'s and are
versioned apart; errors, strides and streams go through ``_lib``.  Here too is
the scratch that their calls take.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Dict, List, Optional

import torch

from latentserve_amd import _lib

_VP = ctypes.c_void_p
_I64P = ctypes.POINTER(ctypes.c_int64)
_I32 = ctypes.c_int
_F32 = ctypes.c_float
_I64 = ctypes.c_int64
_SZ = ctypes.c_size_t

ABI_VERSION = 1

_SIGNATURES = {
    "ls_serving_abi_version": [],
    "ls_int4_write": [_VP, _I64P, _VP, _I64P, _VP, _VP, _VP, _VP, _VP, _I64P, _I64, _I32, _I32,
                      _I32, _I32, _I32, _VP],
    "ls_int4_read": [_VP, _VP, _VP, _VP, _I64P, _I64, _VP, _I64, _I32, _VP, _VP, _VP, _I32, _I32,
                     _I32, _I32, _I32, _VP],
    "ls_int4_decode_groups": [_I32, _I32, _I32, _I32],
    "ls_int4_decode_workspace_bytes": [_I32, _I32, _I32],
    "ls_int4_decode_counter_ints": [_I32, _I32],
    "ls_paged_decode_int4": [_VP, _I64P, _VP, _VP, _VP, _VP, _I64P, _I64, _VP, _I64, _I32, _VP,
                             _VP, _I64P, _VP, _SZ, _VP, _I32, _I32, _I32, _I32, _I32, _I32, _F32,
                             _VP],
    "ls_page_copy": [_VP, _VP, _VP, _I32, _I64, _VP, _VP, _I32, _VP],
    "ls_token_logprobs_workspace_bytes": [_I32, _I32, _I32],
    "ls_token_logprobs_counter_ints": [_I32, _I32, _I32],
    "ls_token_logprobs": [_VP, _I64, _I32, _VP, _I64, _VP, _VP, _VP, _VP, _VP, _SZ, _VP, _I32,
                          _I32, _I32, _VP],
}

_bound: Optional[ctypes.CDLL] = None


def exported_symbols() -> List[str]:
    return sorted(_SIGNATURES)


def lib() -> ctypes.CDLL:
    """The library with this header's entry points bound.  Raises
    HipLibraryMissing where it has none or another version's."""
    global _bound
    handle = _lib.lib()
    if handle is not _bound:
        if not isinstance(handle, ctypes.CDLL):      # (a stand-in has its own signatures)
            return handle
        version = getattr(handle, "ls_serving_abi_version", None)
        got = None if version is None else version()
        if got != ABI_VERSION:
            raise _lib.HipLibraryMissing(
                f"{_lib.LIB_PATH} has version {got} of latentserve_amd_serving.h, this binding "
                f"expects {ABI_VERSION}: rebuild it with `python -m latentserve_amd.csrc.build`")
        for name, argtypes in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.argtypes = argtypes
            fn.restype = _SZ if name.endswith(("_bytes", "_ints")) else _I32
        _bound = handle
    return handle


# Arrival counters (int32, zero at rest: every call leaves its own at zero).
# Two calls that may run at once may not share them: a device's streams have one
# buffer each, and a call recorded into a graph, which may be replayed beside
# anything, has a slice of its own for good.  Slices come from zero-filled slabs
# made outside captures; a capture that finds none left has its counters
# zeroed by the graph itself.
_SLAB_INTS = 1 << 18
_by_stream: Dict[tuple, torch.Tensor] = {}
_slabs: Dict[int, List] = {}          # device index -> [newest slab, ints taken]
_kept: List[torch.Tensor] = []        # slabs and outgrown buffers: graphs may hold their addresses


def _slab(device: torch.device) -> None:
    slab = torch.zeros(_SLAB_INTS, dtype=torch.int32, device=device)
    # (the fill is on this stream; a graph that takes a slice may replay on any)
    torch.cuda.current_stream(device).synchronize()
    _kept.append(slab)
    _slabs[device.index] = [slab, 0]


# (what torch.cuda.is_current_stream_capturing and current_device wrap, without their
# checks that CUDA is initialised: a launch's stream lookup has done that)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_NOTHING = contextlib.nullcontext()


def counters(device: torch.device, stream: int, ints: int) -> torch.Tensor:
    """At least `ints` zeroed counters for one call on `stream` of `device`."""
    index = device.index
    have = _slabs.get(index)
    if _capturing():
        take = -(-ints // 32) * 32                       # whole 128-byte lines
        if have is None or have[1] + take > _SLAB_INTS:
            return torch.zeros(ints, dtype=torch.int32, device=device)
        at = have[1]
        have[1] += take
        return have[0][at:at + take]
    if have is None or 2 * have[1] > _SLAB_INTS:         # room for the captures to come
        _slab(device)
    buf = _by_stream.get((index, stream))
    if buf is None or buf.numel() < ints:
        if buf is not None:
            _kept.append(buf)
        buf = torch.zeros(max(ints, 4096), dtype=torch.int32, device=device)
        _by_stream[index, stream] = buf
    return buf


def on(device: torch.device):
    """`device` as the current one for a launch (nothing to do where it is)."""
    return _NOTHING if device.index == _current_device() else torch.cuda.device(device)
