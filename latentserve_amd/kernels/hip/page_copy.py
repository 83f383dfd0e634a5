"""Pages copied to other pages of the same pools on a HIP kernel.

What branching a sequence (its last, partly filled page) and compacting a cache
need: every layer's K and V pools, scales and bounds in one launch, the page
numbers in the launch's arguments.
"""

from __future__ import annotations

import operator
import struct
from array import array
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
        src, dst = array("i", src), array("i", dst)
    except (TypeError, OverflowError):
        raise ValueError("page numbers must be whole numbers on the host, below 2^31") from None
    n = len(src)
    if len(dst) != n:
        raise ValueError(f"{n} source pages for {len(dst)} destinations")
    if not tensors:
        return
    first = tensors[0]
    dev = first.device
    count, pages = len(tensors), first.shape[0] if first.dim() else 0
    if set(map(_length, tensors)) != {pages}:
        raise ValueError(f"every tensor must have {pages} pages, got "
                         f"{[tuple(t.shape) for t in tensors][:8]}")
    if set(map(torch.Tensor.get_device, tensors)) != {first.get_device()}:
        raise ValueError("the tensors must be on one device")
    if torch.is_grad_enabled() and any(map(_requires_grad, tensors)):
        raise ValueError("a page copy records no gradient")
    if all(map(torch.Tensor.is_contiguous, tensors)):
        sizes = steps = [b // pages if pages else 0 for b in map(_nbytes, tensors)]
    else:
        steps, sizes = _layouts(tensors)
    stream = _lib.stream_of(dev)
    if n == 0:
        return
    ptrs = list(map(torch.Tensor.data_ptr, tensors))
    if 0 in sizes:
        keep = [i for i in range(count) if sizes[i]]
        ptrs, steps, sizes = ([a[i] for i in keep] for a in (ptrs, steps, sizes))
        count = len(keep)
    if dev.index != _serving.current_device():
        with torch.cuda.device(dev):
            return copy_pages(tensors, src, dst)
    int64s = struct.Struct(f"{count}q").pack
    size = int64s(*sizes)
    rc = _serving.lib().ls_page_copy(int64s(*ptrs), size if steps is sizes else int64s(*steps), size,
                                     count, pages, _address(src), _address(dst), n, stream)
    _lib.check(rc, "ls_page_copy")


# (the C slot, past len()'s Python wrapper: a tensor without dimensions has 0)
_length = torch._C.TensorBase.__len__
_nbytes = operator.attrgetter("nbytes")
_requires_grad = operator.attrgetter("requires_grad")


def _address(a: array) -> int:
    return a.buffer_info()[0]


def _layouts(tensors):
    """Bytes from page to page, and of a page, of tensors that are not all contiguous."""
    steps, sizes = [], []
    for t in tensors:
        elems, st = 1, t.stride()
        for k in range(t.dim() - 1, 0, -1):
            if t.shape[k] != 1 and st[k] != elems and t.numel():
                raise ValueError("a page's elements must be contiguous")
            elems *= t.shape[k]
        steps.append(st[0] * t.element_size())
        sizes.append(elems * t.element_size())
    return steps, sizes
