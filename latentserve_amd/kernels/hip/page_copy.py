"""Pages copied to other pages of the same pools on a HIP kernel.

What branching a sequence (its last, partly filled page) and compacting a cache
need: every layer's K and V pools, scales and bounds in one launch, the page
numbers in the launch's arguments.
"""

from __future__ import annotations

import ctypes
import operator
from typing import Sequence

import torch

from latentserve_amd import _lib, _serving


def copy_pages(tensors: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """t[dst[i]] = t[src[i]] for every t of `tensors` and every i: a bit-exact copy.

    The tensors share their first dimension (the pages) and device; a page's
    elements are contiguous, its distance to the next is free.  src and dst are
    page numbers on the host (a graph that records the call keeps them).  A page
    may be copied to several; one that is written twice, or both read and written,
    is refused, and then nothing is copied.  Tensors that overlap are the
    caller's to avoid."""
    try:
        if any(isinstance(p, torch.Tensor) and p.device.type != "cpu" for p in (src, dst)):
            raise TypeError
        src, dst = (list(map(operator.index, p)) for p in (src, dst))
    except TypeError:
        raise ValueError("page numbers must be whole numbers on the host") from None
    n = len(src)
    if len(dst) != n:
        raise ValueError(f"{n} source pages for {len(dst)} destinations")
    if not tensors:
        return
    first = tensors[0]
    pages, dev = first.shape[0] if first.dim() else 0, first.device
    count = len(tensors)
    ptrs, steps, sizes = ((ctypes.c_int64 * count)() for _ in range(3))
    for i, t in enumerate(tensors):
        if t.dim() == 0 or t.shape[0] != pages:
            raise ValueError(f"every tensor must have {pages} pages, got {tuple(t.shape)}")
        if t.device != dev:
            raise ValueError("the tensors must be on one device")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("a page copy records no gradient")
        elems = 1
        st = t.stride()
        for k in range(t.dim() - 1, 0, -1):
            if t.shape[k] != 1 and st[k] != elems and t.numel():
                raise ValueError("a page's elements must be contiguous")
            elems *= t.shape[k]
        size = t.element_size()
        ptrs[i], steps[i], sizes[i] = t.data_ptr(), st[0] * size, elems * size
    stream = _lib.stream_of(dev)
    if n == 0:
        return
    if min(min(src), min(dst)) < 0 or max(max(src), max(dst)) >= pages:
        raise ValueError(f"page numbers must be in [0, {pages})")      # (before 32 bits wrap them)
    if any(size == 0 for size in sizes):
        keep = [i for i in range(count) if sizes[i]]
        ptrs, steps, sizes = ((ctypes.c_int64 * len(keep))(*(a[i] for i in keep))
                              for a in (ptrs, steps, sizes))
        count = len(keep)
    with _serving.on(dev):
        rc = _serving.lib().ls_page_copy(ctypes.cast(ptrs, ctypes.c_void_p), steps, sizes, count,
                                         pages, (ctypes.c_int32 * n)(*src),
                                         (ctypes.c_int32 * n)(*dst), n, stream)
    _lib.check(rc, "ls_page_copy")
