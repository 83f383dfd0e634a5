"""4-bit paged K/V pools on HIP kernels: write, read back, decode attention.

The KV cache in a quarter of the fp16 pools' bytes (160 a token and KV head
instead of 512).  Unlike the INT8 pools a token's entry depends on that token
alone, so there is no last-page residual: pages can be shared, copied and
rewound at any token.

Per (token, head), each group of 32 adjacent channels has a minimum m and a step
s = fp16((max - m) / 15) (the next smaller one where m + 15 s would pass fp16's
largest value), both fp16; a channel's code is the whole number nearest
to (x - m) / s (ties to even) in 0..15 and stands for fp16(m + s * code).

``Int4Pools`` holds the four tensors of a layer:

    k_codes   uint8 [nb, H, 16, 64]      k_affine  fp16 [nb, H, 16, 4, 2]
    v_codes   uint8 [nb, H, 16, 16, 4]   v_affine  fp16 [nb, H, 4, 4, 2, 4]

(include/latentserve_amd_serving.h says where each channel lies).  A page's heads
are contiguous; from page to page any stride of whole 16 bytes will do, so the
pools of several layers may share one allocation.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from latentserve_amd import _lib, _serving

HEAD_DIM = 128
PAGE = 16
GROUP = 32
MAX_NREP = 16
_MAX_WIDTH = 1 << 24            # pages of a block table
_SCALE = 1.0 / math.sqrt(HEAD_DIM)

_SHAPES = ((PAGE, 64), (PAGE, 4, 2), (16, PAGE, 4), (4, 4, 2, 4))
_INNER = ((64, 1), (8, 2, 1), (64, 4, 1), (32, 8, 4, 1))
_HEAD = (1024, 128, 1024, 128)          # elements of one head's part of a page
_DTYPES = (torch.uint8, torch.float16, torch.uint8, torch.float16)


class Int4Pools(NamedTuple):
    k_codes: torch.Tensor
    k_affine: torch.Tensor
    v_codes: torch.Tensor
    v_affine: torch.Tensor


def empty_pools(num_blocks: int, kv_heads: int, device) -> Int4Pools:
    """Zeroed pools of num_blocks pages (every entry stands for 0)."""
    return Int4Pools(*(torch.zeros((num_blocks, kv_heads) + s, dtype=d, device=device)
                       for s, d in zip(_SHAPES, _DTYPES)))


_STEPS: dict = {}               # contiguous pools' page strides by their heads


def _pools(pools, written: bool = False):
    """(num_blocks, heads, C arguments) of checked pools."""
    try:
        kc, ka, vc, va = pools
    except (TypeError, ValueError):
        raise ValueError("4-bit pools are (k_codes, k_affine, v_codes, v_affine)") from None
    nb, h = kc.shape[:2]
    if kc.dtype is vc.dtype is torch.uint8 and ka.dtype is va.dtype is torch.float16 \
            and kc.shape == (nb, h, PAGE, 64) and ka.shape == (nb, h, PAGE, 4, 2) \
            and vc.shape == (nb, h, 16, PAGE, 4) and va.shape == (nb, h, 4, 4, 2, 4) \
            and kc.is_contiguous() and ka.is_contiguous() and vc.is_contiguous() \
            and va.is_contiguous() \
            and kc.get_device() == ka.get_device() == vc.get_device() == va.get_device():
        steps = _STEPS.get(h)
        if steps is None:
            steps = _STEPS[h] = _lib._I64N[4](h * 1024, h * 256, h * 1024, h * 256)
        return nb, h, (kc.data_ptr(), ka.data_ptr(), vc.data_ptr(), va.data_ptr(), steps, nb)
    return _uncommon_pools(pools, written)


def _uncommon_pools(pools, written: bool):
    """The same for pools that are not simply contiguous, or not pools."""
    nb, h = pools[0].shape[:2]
    dev = pools[0].device
    steps = []
    for name, t, shape, inner, head, dtype in zip(Int4Pools._fields, pools, _SHAPES, _INNER, _HEAD,
                                                  _DTYPES):
        st = t.stride()
        if t.dtype != dtype or t.shape != (nb, h) + shape:
            raise ValueError(f"{name} must be {dtype} {(nb, h) + shape}, got {t.dtype} "
                             f"{tuple(t.shape)}")
        if t.device != dev:
            raise ValueError("the pools must be on one device")
        if st[2:] != inner or (h > 1 and st[1] != head):
            raise ValueError(f"{name}: a page's heads must be contiguous")
        if written and nb > 1 and st[0] < h * head:
            raise ValueError(f"{name}: pages that overlap cannot be written")
        steps.append(st[0] * t.element_size())
    return nb, h, (*(t.data_ptr() for t in pools), _lib._I64N[4](*steps), nb)


def _rows(name: str, t: torch.Tensor):
    """The strides of checked rows [., ., ., 128]; a dimension of one row has none that
    matters."""
    if t.dtype is not torch.float16:
        raise ValueError(f"{name} must be float16, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which a 4-bit cache does not carry")
    s0, s1, s2, unit = t.stride()
    n0, n1, n2, _ = t.shape
    s0, s1, s2 = (s0 if n0 > 1 else 0), (s1 if n1 > 1 else 0), (s2 if n2 > 1 else 0)
    if unit != 1 or t.data_ptr() & 15 or (s0 | s1 | s2) & 7:
        raise ValueError(f"{name} rows must be 16-byte aligned and unit-stride")
    return _lib._I64N[3](s0, s1, s2)


def _span(t: torch.Tensor):
    """First byte of t and the one behind its last (the gaps between rows included)."""
    last = sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, b: int, device: int) -> None:
    if block_tables.dtype is not torch.int32 or seq_lens.dtype is not torch.int32 \
            or block_tables.dim() != 2 or seq_lens.shape != (b,) or block_tables.stride(1) != 1 \
            or (b > 1 and seq_lens.stride(0) != 1):
        raise ValueError("block tables [B, pages] and sequence lengths [B] must be unit-stride "
                         f"int32, of {b} sequences")
    if block_tables.shape[0] != b:
        raise ValueError(f"block tables must have {b} rows")
    if block_tables.get_device() != device or seq_lens.get_device() != device:
        raise ValueError("block tables and sequence lengths must be on the pools' device")


# Launch sizes by a decode's shape: (groups, workspace bytes, counters).
_SIZES: dict = {}


def _sizes(b: int, h: int, n_rep: int, width: int, bound: int):
    key = (b, h, n_rep, width, bound)
    got = _SIZES.get(key)
    if got is None:
        if width > _MAX_WIDTH:
            raise ValueError(f"block tables of {width} pages are too wide")
        lib = _serving.lib()
        groups = lib.ls_int4_decode_groups(b, h, width, bound)
        got = (groups, lib.ls_int4_decode_workspace_bytes(groups, h, n_rep),
               lib.ls_int4_decode_counter_ints(groups, h))
        if len(_SIZES) >= 4096:
            _SIZES.clear()
        _SIZES[key] = got
    return got


def write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, pools) -> None:
    """k, v [B, H, n, 128] fp16 (any strides of whole 16 bytes) quantized into flat
    token slots [B * n] int64 (block * 16 + offset; outside the pool: not
    written).  Slots are distinct.  Other tokens keep their entries.  A group of 32
    channels that holds a NaN or an infinity reads back as NaN."""
    nb, h, args = _pools(pools, written=True)
    dev = pools[0].device
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[1] != h or shape[3] != HEAD_DIM:
        raise ValueError(f"k and v must be [B, {h}, n, {HEAD_DIM}], got {tuple(shape)} and "
                         f"{tuple(v.shape)}")
    b, _, n, _ = shape
    if slots.dtype is not torch.int64 or slots.shape != (b * n,) \
            or (b * n > 1 and slots.stride(0) != 1):
        raise ValueError(f"slots must be {b * n} unit-stride int64 values")
    index = pools[0].get_device()
    if k.get_device() != index or v.get_device() != index or slots.get_device() != index:
        raise ValueError("k, v and slots must be on the pools' device")
    stream = _lib.stream_of(dev)
    if b * n == 0:
        return
    ks, vs = _rows("k", k), _rows("v", v)
    if index != _serving.current_device():
        with torch.cuda.device(index):
            return write(k, v, slots, pools)
    rc = _serving.lib().ls_int4_write(k.data_ptr(), ks, v.data_ptr(), vs, slots.data_ptr(), *args,
                                      b, h, n, HEAD_DIM, PAGE, stream)
    _lib.check(rc, "ls_int4_write")


def read(pools, block_tables: torch.Tensor, seq_lens: torch.Tensor,
         length: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [B, H, length, 128] fp16: the values that each sequence's first
    `length` entries stand for (default: the table's width), zeros past its
    end.  Token-major in memory, as [B, length, H, 128]."""
    nb, h, args = _pools(pools)
    dev = pools[0].device
    b = block_tables.shape[0]
    _tables(block_tables, seq_lens, b, pools[0].get_device())
    length = block_tables.shape[1] * PAGE if length is None else int(length)
    if length < 0:
        raise ValueError(f"length must be >= 0, got {length}")
    stream = _lib.stream_of(dev)
    if dev.index != _serving.current_device():
        with torch.cuda.device(dev):
            return read(pools, block_tables, seq_lens, length)
    width = block_tables.shape[1]
    if width > _MAX_WIDTH:
        raise ValueError(f"block tables of {width} pages are too wide")
    token = h * HEAD_DIM
    shape, steps = (b, h, length, HEAD_DIM), (length * token, HEAD_DIM, token, 1)
    k = torch.empty_strided(shape, steps, dtype=torch.float16, device=dev)
    v = torch.empty_strided(shape, steps, dtype=torch.float16, device=dev)
    if width == 0:
        return k.zero_(), v.zero_()
    if b * length:
        rc = _serving.lib().ls_int4_read(
            *args, block_tables.data_ptr(), block_tables.stride(0), width, seq_lens.data_ptr(),
            k.data_ptr(), v.data_ptr(), b, h, HEAD_DIM, PAGE, length, stream)
        _lib.check(rc, "ls_int4_read")
    return k, v


def paged_decode_int4(q: torch.Tensor, pools, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                      max_seq_len: Optional[int] = None, softmax_scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention over 4-bit pools: q [B, H, n_rep, 128] fp16, n_rep 1..16 ->
    a new tensor of its shape, or `out`.

    max_seq_len: the longest sequence expected (a graph's bucket); it only sizes
    the launch, a longer one is attended whole.  Sequences of no tokens give
    zeros, and blocks outside the pool are skipped.  out may not overlap q.  Each
    call has its own scratch, so calls may run at once on several streams and from
    several graphs.  Sums are fp32, of weights of 21 bits and more; their order may differ
    from call to call, and the result by a rounding."""
    _, h, args = _pools(pools)
    shape, dev, index = q.shape, q.device, q.get_device()
    if len(shape) != 4 or shape[1] != h or shape[3] != HEAD_DIM \
            or not 1 <= shape[2] <= MAX_NREP:
        raise ValueError(f"q must be [B, {h}, n_rep 1..{MAX_NREP}, {HEAD_DIM}], got "
                         f"{tuple(shape)}")
    if index != pools[0].get_device():
        raise ValueError("q must be on the pools' device")
    b, _, n_rep, _ = shape
    _tables(block_tables, seq_lens, b, index)
    stream = _lib.stream_of(dev)
    qs = _rows("q", q)
    if out is None:
        out = torch.empty(b, h, n_rep, HEAD_DIM, dtype=torch.float16, device=dev)
        os = _lib._I64N[3](h * n_rep * HEAD_DIM, n_rep * HEAD_DIM, HEAD_DIM)
    else:
        if out.shape != shape or out.device != dev:
            raise ValueError(f"out must be {tuple(shape)} on {dev}")
        os = _rows("out", out)
        if b and _span(out)[0] < _span(q)[1] and _span(q)[0] < _span(out)[1]:
            raise ValueError("out may not overlap q, which other workgroups still read")
    if index != _serving.current_device():
        with torch.cuda.device(dev):
            return paged_decode_int4(q, pools, block_tables, seq_lens, max_seq_len, softmax_scale,
                                     out)
    width = block_tables.shape[1]
    if b == 0 or width == 0:
        return out.zero_()
    groups, nbytes, ints = _sizes(b, h, n_rep, width,
                                  0 if max_seq_len is None else max(1, int(max_seq_len)))
    scale = _SCALE if softmax_scale is None else float(softmax_scale)
    work, cnt = _serving.scratch(dev, stream, nbytes, ints)
    rc = _serving.lib().ls_paged_decode_int4(
        q.data_ptr(), qs, *args, block_tables.data_ptr(), block_tables.stride(0), width,
        seq_lens.data_ptr(), out.data_ptr(), os, work.data_ptr(), nbytes, cnt.data_ptr(), b, h,
        n_rep, HEAD_DIM, PAGE, groups, scale, stream)
    _lib.check(rc, "ls_paged_decode_int4")
    return out
