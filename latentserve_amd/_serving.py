"""ctypes binding of the second header, include/latentserve_amd_serving.h: the 4-bit
paged cache, page copies and token log probabilities.

The entry points live in the same liblatentserve_hip.so as ``_lib``'s and are
versioned apart; errors, strides and streams go through ``_lib``.  Here too is
the scratch that their calls take.
"""

from __future__ import annotations

import contextlib
import ctypes
import threading
import weakref
from collections import deque
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


# Scratch of a call: records (any contents) and arrival counters (int32, zero at rest:
# every call leaves its own at zero).  Two calls that may run at once may not share
# it.  A device's streams have their own, kept and grown up to a bound (a stream is
# known by its handle, as to torch's allocator: work of a destroyed stream has ended
# before its handle is used again).  A call recorded into a graph, which may be
# replayed beside anything, has records of the graph's own and a slice of counters
# that goes back when the graph is gone (counters_of), or is the call's for good where
# nobody says which graph that is.  Slices come from zero-filled slabs made
# outside captures; a capture that finds none left has its counters zeroed by the
# graph itself.
_SLAB_INTS = 1 << 20                  # (a full decode takes 2048: over 250 layers captured at once)
_KEPT_BYTES, _KEPT_INTS = 16 << 20, 1 << 18          # a larger call's go back to the allocator
_by_stream: Dict[tuple, tuple] = {}   # (device index, stream) -> (records, counters)
_slabs: Dict[int, List] = {}          # device index -> [newest slab, ints taken]
_kept: List[torch.Tensor] = []        # slabs, whose addresses graphs hold
_free: Dict[tuple, List] = {}         # (device index, ints) -> slices that no graph holds
_returned: deque = deque()            # (device index, slices) of graphs that are gone
_owner = threading.local()            # .slices: where this thread's captured calls list theirs
_lock = threading.Lock()              # two captures at once may not get one slice
# (what torch.cuda.is_current_stream_capturing and current_device wrap, without their
# checks that CUDA is initialised: a launch's stream lookup has done that)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)
current_device = getattr(torch._C, "_cuda_getDevice", None)


def _room(device: torch.device) -> None:
    """A slab with room for the captures to come."""
    have = _slabs.get(device.index)
    if have is None or 2 * have[1] > _SLAB_INTS:
        slab = torch.zeros(_SLAB_INTS, dtype=torch.int32, device=device)
        # (filled on this stream; a graph that takes a slice may replay on any)
        torch.cuda.current_stream(device).synchronize()
        _kept.append(slab)
        _slabs[device.index] = [slab, 0]


@contextlib.contextmanager
def counters_of(graph: torch.cuda.CUDAGraph):
    """Around a capture: the counters that its calls take go back once `graph` is gone.

        with counters_of(g), torch.cuda.graph(g):
            ...
    """
    index = torch.cuda.current_device()
    if not _capturing():                                     # (entered inside it: later captures)
        _recycle()
        _room(torch.device("cuda", index))
    outer, _owner.slices = getattr(_owner, "slices", None), []
    try:
        yield
    finally:
        slices, _owner.slices = _owner.slices, outer
        if slices:
            # (a finalizer may run anywhere, under the lock too: it takes none)
            weakref.finalize(graph, _returned.append, (index, slices)).atexit = False


def _recycle() -> None:
    """The slices of graphs that are gone become free ones."""
    gone = []
    while True:
        try:
            gone.append(_returned.popleft())
        except IndexError:
            break
    for i in {i for i, _ in gone}:
        torch.cuda.synchronize(i)            # (a graph may be dropped while its last replay runs)
    with _lock:
        for i, slices in gone:
            for cnt in slices:
                _free.setdefault((i, cnt.numel()), []).append(cnt)


def _captured_scratch(device: torch.device, nbytes: int, ints: int):
    work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    cnt = _slice_for_capture(device.index, ints)
    return work, torch.zeros(ints, dtype=torch.int32, device=device) if cnt is None else cnt


def _slice_for_capture(index: int, ints: int) -> Optional[torch.Tensor]:
    take = -(-ints // 32) * 32                               # whole 128-byte lines
    with _lock:
        cnt = _slice(index, take)
    slices = getattr(_owner, "slices", None)
    if cnt is not None and slices is not None:
        slices.append(cnt)
    return cnt


def _slice(index: int, take: int) -> Optional[torch.Tensor]:
    free = _free.get((index, take))
    if free:
        return free.pop()
    have = _slabs.get(index)
    if have is None or have[1] + take > _SLAB_INTS:
        return None
    at = have[1]
    have[1] += take
    return have[0][at:at + take]


def scratch(device: torch.device, stream: int, nbytes: int, ints: int):
    """(records, counters) tensors of at least these sizes for one call on `stream`, the
    current one of the current device."""
    if _capturing():
        return _captured_scratch(device, nbytes, ints)
    index = device.index
    have = _slabs.get(index)
    if have is None or 2 * have[1] > _SLAB_INTS:
        _room(device)
    got = _by_stream.get((index, stream))
    if got is None or got[0].numel() < nbytes or got[1].numel() < ints:
        if nbytes > _KEPT_BYTES or ints > _KEPT_INTS:
            return (torch.empty(nbytes, dtype=torch.uint8, device=device),
                    torch.zeros(ints, dtype=torch.int32, device=device))
        # (an outgrown pair goes back to the allocator, which hands it on in this
        # stream's order)
        old = got or (torch.empty(0, dtype=torch.uint8), torch.empty(0, dtype=torch.int32))
        got = (torch.empty(max(nbytes, old[0].numel(), 1 << 16), dtype=torch.uint8, device=device),
               torch.zeros(max(ints, old[1].numel(), 4096), dtype=torch.int32, device=device))
        _by_stream[index, stream] = got
    return got
