"""ctypes binding of the third header, include/latentserve_amd_tree.h: attention of
drafted trees, accepted paths, weight sums and eviction.

The entry points live in the same liblatentserve_hip.so as ``_lib``'s and are
versioned apart; errors, strides and streams go through ``_lib``, scratch through
``_serving``.
"""

from __future__ import annotations

import ctypes
import functools
import operator
from array import array as Array
from typing import List, Optional

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
    "ls_tree_abi_version": [],
    "ls_tree_masks": [_VP, _VP, _VP, _I32, _I32, _VP],
    "ls_tree_attention_workspace_bytes": [_I32, _I32, _I32, _I32, _I32, _I32],
    "ls_tree_attention": [_VP, _I64P, _VP, _VP, _I64P, _I64, _VP, _I64, _I32, _VP, _VP, _VP, _VP,
                          _I64P, _VP, _VP, _SZ, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _F32,
                          _VP],
    "ls_decode_weights_workspace_bytes": [_I32, _I32, _I32, _I32, _I32],
    "ls_paged_decode_weights": [_VP, _I64P, _VP, _VP, _I64P, _I64, _VP, _I64, _I32, _VP, _VP,
                                _I64P, _VP, _I64P, _I64, _VP, _I32, _VP, _SZ, _I32, _I32, _I32,
                                _I32, _I32, _I32, _F32, _VP],
    "ls_add_weights": [_VP, _I64P, _VP, _VP, _I64P, _I64, _VP, _I64, _I32, _VP, _VP, _I64P, _I64,
                       _VP, _I32, _VP, _VP, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _I32, _F32,
                       _VP],
    "ls_accept_tokens": [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I32, _I64P, _I64, _VP, _I64,
                         _I32, _VP, _I32, _I32, _I32, _I32, _I32, _VP],
    "ls_select_tokens": [_VP, _I64P, _I64, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _I32, _I32, _VP],
    "ls_move_tokens": [_VP, _VP, _I32, _I64P, _I64, _VP, _I64, _I32, _VP, _VP, _I32, _I32, _I32,
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
        version = getattr(handle, "ls_tree_abi_version", None)
        got = None if version is None else version()
        if got != ABI_VERSION:
            raise _lib.HipLibraryMissing(
                f"{_lib.LIB_PATH} has version {got} of latentserve_amd_tree.h, this binding "
                f"expects {ABI_VERSION}: rebuild it with `python -m latentserve_amd.csrc.build`")
        for name, argtypes in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.argtypes = argtypes
            fn.restype = _SZ if name.endswith("_bytes") else _I32
        _bound = handle
    return handle


# ---- checks that the entry points share -------------------------------------------

HEAD_DIM = 128
PAGE = 16
MAX_NREP = 16
MAX_NODES = 256
_MAX_WIDTH = 1 << 24            # pages of a block table
_MAX_TOKEN_STRIDE = 1 << 24     # elements


_STRIDES: dict = {}             # contiguous rows' strides by their shapes


def whole_rows(shape: torch.Size):
    """The strides of contiguous rows of a shape [..., 128], as C int64."""
    got = _STRIDES.get(shape)
    if got is None:
        st = [HEAD_DIM]
        for n in shape[-2:0:-1]:
            st.insert(0, st[0] * n)
        if len(_STRIDES) >= 4096:
            _STRIDES.clear()
        got = _STRIDES[shape] = _lib._I64N[len(st)](*st)
    return got


def rows(name: str, t: torch.Tensor):
    """The strides of checked rows [..., 128]; a dimension of one row has none that
    matters."""
    if t.dtype is not torch.float16:
        raise ValueError(f"{name} must be float16, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which a cache's attention does not record")
    if t.is_contiguous() and not t.data_ptr() & 15:
        return whole_rows(t.shape)
    *st, unit = t.stride()
    st = [s if n > 1 else 0 for s, n in zip(st, t.shape)]
    bits = t.data_ptr()
    for s in st:
        bits |= 2 * s
    if unit != 1 or bits & 15:
        raise ValueError(f"{name} rows must be 16-byte aligned and unit-stride")
    return _lib._I64N[len(st)](*st)


_PLACES: dict = {}              # contiguous pools' strides by their heads


def pool(name: str, t: torch.Tensor):
    """(heads, blocks, strides as C int64) of a checked pool [nb, 16, H, 128]."""
    shape = t.shape
    if t.dtype is not torch.float16 or len(shape) != 4 or shape[1] != PAGE \
            or shape[3] != HEAD_DIM or not shape[0] or not shape[2]:
        raise ValueError(f"{name} must be float16 [num_blocks, {PAGE}, H, {HEAD_DIM}], got {t.dtype} "
                         f"{tuple(shape)}")
    h = shape[2]
    if t.is_contiguous() and not t.data_ptr() & 15:
        got = _PLACES.get(h)
        if got is None:
            got = _PLACES[h] = _lib._I64N[3](PAGE * h * HEAD_DIM, h * HEAD_DIM, HEAD_DIM)
        return h, shape[0], got
    sb, st, sh, unit = t.stride()
    if unit != 1 or (2 * (sb | st | sh) | t.data_ptr()) & 15 or st > _MAX_TOKEN_STRIDE:
        raise ValueError(f"{name} rows must be 16-byte aligned and unit-stride, tokens at most "
                         f"{_MAX_TOKEN_STRIDE} elements apart")
    return h, shape[0], _lib._I64N[3](sb, st, sh)


def two_pools(k_pool: torch.Tensor, v_pool: torch.Tensor):
    h, nb, steps = pool("k_pool", k_pool)
    if v_pool.shape != k_pool.shape or v_pool.dtype is not torch.float16 \
            or v_pool.stride() != k_pool.stride() or v_pool.data_ptr() & 15:
        raise ValueError(f"v_pool must be alike, float16 {tuple(k_pool.shape)} with the same strides")
    if v_pool.get_device() != k_pool.get_device():
        raise ValueError("the pools must be on one device")
    return h, nb, steps


def tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, b: int, device: int) -> int:
    """The width of checked tables of b sequences."""
    if block_tables.dtype is not torch.int32 or seq_lens.dtype is not torch.int32 \
            or block_tables.dim() != 2 or block_tables.shape[0] != b or seq_lens.shape != (b,) \
            or block_tables.stride(1) != 1 or (b > 1 and seq_lens.stride(0) != 1):
        raise ValueError("block tables [B, pages] and sequence lengths [B] must be unit-stride "
                         f"int32, of {b} sequences")
    if block_tables.get_device() != device or seq_lens.get_device() != device:
        raise ValueError("block tables and sequence lengths must be on the pools' device")
    width = block_tables.shape[1]
    if width > _MAX_WIDTH:
        raise ValueError(f"block tables of {width} pages are too wide")
    return width


def whole(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int) -> int:
    """The address of a checked contiguous tensor."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the pools' device")
    return t.data_ptr()


def span(t: torch.Tensor):
    """First byte of t and the one behind its last (the gaps between rows included)."""
    last = sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def rows_apart(t: torch.Tensor) -> bool:
    """Whether each stride of rows [..., 128] clears what the smaller ones span, in whatever
    order the dimensions lie (a dimension of one has none that matters)."""
    end = HEAD_DIM
    for st, n in sorted(zip(t.stride()[:-1], t.shape[:-1])):
        if n > 1:
            if st < end:
                return False
            end += st * (n - 1)
    return True


def apart(name: str, out: torch.Tensor, q: torch.Tensor) -> None:
    if not out.is_contiguous() and not rows_apart(out):
        raise ValueError(f"{name} may not have rows that overlap or interleave: got strides "
                         f"{out.stride()} of {tuple(out.shape)}")
    if out.numel() and q.numel():
        (a, b), (c, d) = span(out), span(q)
        if a < d and c < b:
            raise ValueError(f"{name} may not overlap q, which other workgroups still read")


_FP16 = {torch.float16}


def pool_lists(k_pools, v_pools):
    """(heads, blocks, strides, device, two C arrays of addresses) of checked layers' pools
    that are written to."""
    n = len(k_pools)
    if n != len(v_pools):
        raise ValueError(f"{n} K pools for {len(v_pools)} V pools")
    first = k_pools[0]
    h, nb, steps = pool("a pool", first)
    pools = [*k_pools, *v_pools]
    # (an attribute of all at a time: half the host time of a loop over 56 pools)
    at = list(map(torch.Tensor.data_ptr, pools))
    # (contiguous tensors of a size have the same strides, where a stride matters)
    alike = all(map(torch.Tensor.is_contiguous, pools)) if first.is_contiguous() else \
        len(set(map(torch.Tensor.stride, pools))) == 1
    if len(set(map(torch.Tensor.size, pools))) > 1 or not alike \
            or len(set(map(torch.Tensor.get_device, pools))) > 1 \
            or set(map(torch.Tensor.dtype.__get__, pools)) != _FP16 \
            or functools.reduce(operator.or_, at) & 15:
        raise ValueError("the layers' pools must be alike: float16 "
                         f"{tuple(first.shape)}, of the same strides, on one device")
    if len(set(at)) < 2 * n:
        raise ValueError("a pool is listed twice: its rows would be moved twice")
    if not first.is_contiguous() and not rows_apart(first):
        raise ValueError("pools that are written may not have rows that overlap or interleave: got "
                         f"strides {first.stride()} of {tuple(first.shape)}")
    if torch.is_grad_enabled() and any(map(torch.Tensor.requires_grad.__get__, pools)):
        raise ValueError("a move of cached tokens records no gradient")
    array = ctypes.c_void_p * n
    both = (array * 2).from_buffer_copy(Array("Q", at))
    return h, nb, steps, first.device, both[0], both[1]


# Workspace bytes by a call's sizes.
_SIZES: dict = {}


def workspace_bytes(name: str, *sizes: int) -> int:
    key = (name, sizes)
    got = _SIZES.get(key)
    if got is None:
        if max(sizes) >= 1 << 31:                             # (C ints)
            raise ValueError("sizes past 2^31")
        got = getattr(lib(), name)(*sizes)
        if len(_SIZES) >= 4096:
            _SIZES.clear()
        _SIZES[key] = got
    return got


def bound_of(max_seq_len, width: int) -> int:
    """max_seq_len as the C calls take it: at least 1, no larger than the table (0: it)."""
    if max_seq_len is None:
        return 0
    n = int(max_seq_len)
    return 1 if n < 1 else n if n < width * PAGE else 0
