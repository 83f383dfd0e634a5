"""Eviction from the fp16 paged cache by accumulated attention weight, on HIP kernels.

A bounded cache keeps, per layer and KV head, the tokens that attention went to:

    out = paged_decode_weights(q, k_pool, v_pool, tables, lens, sums)   # each step
    add_weights(q, lse, k_pool, tables, lens, sums, path=path, lengths=lengths)
                                                 # after a drafted tree's acceptance
    keep, kept = evict_tokens(sums, k_pools, v_pools, tables, lens, budget)

`sums` holds, per KV head and cached position, the attention weight that the
position has got so far, summed over the head's query rows: fp32 [rows, H, T].
Eviction keeps the first few tokens, the most recent ones and those with the
largest sums, and moves their K and V to the front, in order; keys carry their
rotations, so a token's place in the cache says nothing about its position.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from latentserve_amd import _lib, _serving, _tree

HEAD_DIM, PAGE, MAX_NREP, MAX_NODES = _tree.HEAD_DIM, _tree.PAGE, _tree.MAX_NREP, _tree.MAX_NODES
_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def _sums(sums: torch.Tensor, h: int, b: int, rows: Optional[torch.Tensor], index: int):
    """(address, strides, length, rows' address, rows) of checked weight sums [R, H, T]."""
    if sums.dtype is not torch.float32 or sums.dim() != 3 or sums.shape[1] != h:
        raise ValueError(f"sums must be float32 [rows, {h}, T], got {sums.dtype} "
                         f"{tuple(sums.shape)}")
    r, _, length = sums.shape
    sr, sh, unit = sums.stride()
    (near, count), (far, _) = sorted(((sr, r), (sh, h))) if r > 1 < h else \
        ((sh if h > 1 else sr, h if h > 1 else r), (1 << 62, 0))
    if (length > 1 and unit != 1) or (count > 1 and near < length) or far < near * count:
        raise ValueError("rows of sums must be unit-stride and may not overlap")
    if sums.get_device() != index:
        raise ValueError("sums must be on the pools' device")
    if sums.requires_grad and torch.is_grad_enabled():
        raise ValueError("sums require a gradient, which is not recorded")
    rp = None
    if rows is not None:
        rp = _tree.whole("rows", rows, torch.int32, (b,), index)
    elif r < b:
        raise ValueError(f"sums of {r} rows for {b} sequences")
    return sums.data_ptr(), _lib._I64N[2](sr, sh), length, rp, r


def paged_decode_weights(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                         block_tables: torch.Tensor, seq_lens: torch.Tensor, sums: torch.Tensor,
                         rows: Optional[torch.Tensor] = None, max_seq_len: Optional[int] = None,
                         softmax_scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention that also adds up what it attends to: q [B, H, n_rep, 128] fp16,
    n_rep 1..16 -> a new tensor of its shape, or `out`; and for every cached token

        sums[rows[b], h, t] += sum over the n_rep rows of softmax(q K^T scale)[t]

    sums [R, H, T] fp32; rows [B] int32 (None: 0..B-1) names each sequence's row, all
    different; nothing is added for a row outside [0, R), nor for positions from T on.
    Everything else as in ``tree_attention`` of one node.  The call's scratch holds the
    scores, 4 bytes a query row and token of the tables' width (64 sequences of 32 query
    heads in tables for 128K tokens: 1.07 GB): narrow tables to the pages in use
    where that matters."""
    h, nb, steps = _tree.two_pools(k_pool, v_pool)
    shape, dev, index = q.shape, q.device, q.get_device()
    if len(shape) != 4 or shape[1] != h or shape[3] != HEAD_DIM or not 1 <= shape[2] <= MAX_NREP:
        raise ValueError(f"q must be [B, {h}, n_rep 1..{MAX_NREP}, {HEAD_DIM}], got {tuple(shape)}")
    if index != k_pool.get_device():
        raise ValueError("q must be on the pools' device")
    b, _, n_rep, _ = shape
    width = _tree.tables(block_tables, seq_lens, b, index)
    sp, ss, length, rp, r = _sums(sums, h, b, rows, index)
    qs = _tree.rows("q", q)
    if out is not None:
        if out.shape != shape or out.get_device() != index:
            raise ValueError(f"out must be {tuple(shape)} on {dev}")
        _tree.apart("out", out, q)
        os = _tree.rows("out", out)
    stream = _lib.stream_of(dev)
    if out is None:
        out = torch.empty(shape, dtype=torch.float16, device=dev)
        os = _tree.whole_rows(shape)
    if index != _serving.current_device():
        with torch.cuda.device(dev):
            return paged_decode_weights(q, k_pool, v_pool, block_tables, seq_lens, sums, rows,
                                        max_seq_len, softmax_scale, out)
    if b == 0 or width == 0:
        return out.zero_()
    bound = _tree.bound_of(max_seq_len, width)
    nbytes = _tree.workspace_bytes("ls_decode_weights_workspace_bytes", b, h, n_rep, width, bound)
    work, _ = _serving.scratch(dev, stream, nbytes, 0)
    rc = _tree.lib().ls_paged_decode_weights(
        q.data_ptr(), qs, k_pool.data_ptr(), v_pool.data_ptr(), steps, nb, block_tables.data_ptr(),
        block_tables.stride(0), width, seq_lens.data_ptr(), out.data_ptr(), os, sp, ss, length, rp,
        r, work.data_ptr(), nbytes, b, h, n_rep, HEAD_DIM, PAGE, bound,
        _SCALE if softmax_scale is None else float(softmax_scale), stream)
    _lib.check(rc, "ls_paged_decode_weights")
    return out


def add_weights(q: torch.Tensor, lse: torch.Tensor, k_pool: torch.Tensor,
                block_tables: torch.Tensor, seq_lens: torch.Tensor, sums: torch.Tensor,
                rows: Optional[torch.Tensor] = None, path: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, max_seq_len: Optional[int] = None,
                softmax_scale: Optional[float] = None) -> None:
    """The attention weights of accepted tokens added to sums [R, H, T] (rows as in
    paged_decode_weights), after the attention that gave lse.

    q [B, N, H, n_rep, 128] fp16 and lse [B, N, H, n_rep] fp32 as tree_attention() took
    and gave them.  path [B, P] int32 (P <= N): each sequence's accepted nodes in
    order, of which lengths [B] int32 count (None: P); None: all nodes, a chain.
    The cache has been brought together (accept_tokens()) and shortened: seq_lens [B]
    is the context and the path, whose i-th token lies i behind the context and
    sees everything up to itself.  Nodes outside 0..N-1 and rows of lse -inf add
    nothing.  Paths of up to 32 rows (tokens x n_rep) take the time of reading K once,
    longer ones more (5 tokens of 8 rows: twice it)."""
    h, nb, steps = _tree.pool("k_pool", k_pool)
    shape, dev, index = q.shape, q.device, q.get_device()
    if len(shape) != 5 or shape[2] != h or shape[4] != HEAD_DIM \
            or not 1 <= shape[1] <= MAX_NODES or not 1 <= shape[3] <= MAX_NREP:
        raise ValueError(f"q must be [B, N 1..{MAX_NODES}, {h}, n_rep 1..{MAX_NREP}, {HEAD_DIM}], "
                         f"got {tuple(shape)}")
    if index != k_pool.get_device():
        raise ValueError("q must be on the pools' device")
    b, n, _, n_rep, _ = shape
    width = _tree.tables(block_tables, seq_lens, b, index)
    lp = _tree.whole("lse", lse, torch.float32, (b, n, h, n_rep), index)
    sp, ss, length, rp, r = _sums(sums, h, b, rows, index)
    pp = cp = None
    most = n
    if path is not None:
        if path.dim() != 2 or path.shape[1] > n:
            raise ValueError(f"path must be [{b}, up to {n}], got {tuple(path.shape)}")
        most = path.shape[1]
        pp = _tree.whole("path", path, torch.int32, (b, most), index)
    if lengths is not None:
        cp = _tree.whole("lengths", lengths, torch.int32, (b,), index)
    qs = _tree.rows("q", q)
    stream = _lib.stream_of(dev)
    if b == 0 or width == 0 or most == 0:
        return
    if index != _serving.current_device():
        with torch.cuda.device(dev):
            return add_weights(q, lse, k_pool, block_tables, seq_lens, sums, rows, path, lengths,
                               max_seq_len, softmax_scale)
    rc = _tree.lib().ls_add_weights(
        q.data_ptr(), qs, lp, k_pool.data_ptr(), steps, nb, block_tables.data_ptr(),
        block_tables.stride(0), width, seq_lens.data_ptr(), sp, ss, length, rp, r, pp, cp, b, h, n,
        most, n_rep, HEAD_DIM, PAGE, _tree.bound_of(max_seq_len, width),
        _SCALE if softmax_scale is None else float(softmax_scale), stream)
    _lib.check(rc, "ls_add_weights")


def select_tokens(sums: torch.Tensor, seq_lens: torch.Tensor, budget: int, sinks: int = 4,
                  recent: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which positions to keep: sums [L, B, H, T] fp32, seq_lens [B] int32 -> (keep [L, B,
    H, budget] int32, ascending, -1 behind the last; kept, their sums, fp32, 0
    behind the last).

    A sequence of up to `budget` tokens keeps all.  A longer one keeps `budget`: the
    first `sinks`, the last `recent` (default: a quarter of the budget) and the
    largest sums of the others; equal sums by the lower position, a NaN before all
    numbers.  A sequence is taken to be no longer than T."""
    if sums.dtype is not torch.float32 or sums.dim() != 4 or \
            (sums.shape[3] > 1 and sums.stride(3) != 1):
        raise ValueError(f"sums must be unit-stride float32 [L, B, H, T], got {sums.dtype} "
                         f"{tuple(sums.shape)}")
    layers, b, h, length = sums.shape
    dev, index = sums.device, sums.get_device()
    if seq_lens.dtype is not torch.int32 or seq_lens.shape != (b,) \
            or (b > 1 and seq_lens.stride(0) != 1) or seq_lens.get_device() != index:
        raise ValueError(f"seq_lens must be {b} unit-stride int32 values on the sums' device")
    budget, sinks, recent = budget_of(budget, sinks, recent)
    stream = _lib.stream_of(dev)
    if index != _serving.current_device():
        with torch.cuda.device(dev):
            return select_tokens(sums, seq_lens, budget, sinks, recent)
    keep = torch.empty(layers, b, h, budget, dtype=torch.int32, device=dev)
    kept = torch.empty(layers, b, h, budget, dtype=torch.float32, device=dev)
    if layers * b * h:
        rc = _tree.lib().ls_select_tokens(
            sums.data_ptr(), _lib._I64N[3](*sums.stride()[:3]), length, seq_lens.data_ptr(),
            keep.data_ptr(), kept.data_ptr(), layers, b, h, budget, sinks, recent, stream)
        _lib.check(rc, "ls_select_tokens")
    return keep, kept


def budget_of(budget: int, sinks: int, recent: Optional[int]):
    budget, sinks = int(budget), int(sinks)
    if not 1 <= budget < 1 << 31:
        raise ValueError(f"budget must be in [1, 2^31), got {budget}")
    recent = min(budget // 4, budget - sinks) if recent is None else int(recent)
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"a budget of {budget} does not hold {sinks} first and {recent} recent "
                         "tokens")
    return budget, sinks, recent


def move_tokens(keep: torch.Tensor, k_pools: Sequence[torch.Tensor],
                v_pools: Sequence[torch.Tensor], block_tables: torch.Tensor,
                seq_lens: torch.Tensor) -> None:
    """Rows keep[l, b, h, j] of each sequence become its rows j, in every layer's K and V
    pool ([nb, 16, H, 128] fp16, all alike), for j below min(seq_lens[b], budget).

    keep [L, B, H, budget] int32 as select_tokens() gives it: ascending in each row
    (an order that is not moves some rows twice); negative entries move nothing.
    seq_lens [B] are the lengths before.  What lies behind the kept rows is left
    over.  Different sequences' tables name different blocks: shared pages are
    copied first (the cache's evict() does)."""
    layers = len(k_pools)
    if keep.dim() != 4 or keep.shape[0] != layers or layers != len(v_pools):
        raise ValueError(f"keep must be [{layers}, B, H, budget] for {layers} K and {len(v_pools)} "
                         f"V pools, got {tuple(keep.shape)}")
    if layers == 0:
        return
    lists = _tree.pool_lists(k_pools, v_pools)
    _, b, _, budget = keep.shape
    index = k_pools[0].get_device()
    _tree.whole("keep", keep, torch.int32, (layers, b, lists[0], budget), index)
    width = _tree.tables(block_tables, seq_lens, b, index)
    _lib.stream_of(keep.device)
    if b == 0 or budget == 0 or width == 0:
        return
    if index != _serving.current_device():
        with torch.cuda.device(keep.device):
            return _move(keep, lists, block_tables, seq_lens)
    _move(keep, lists, block_tables, seq_lens)


def _move(keep: torch.Tensor, lists, block_tables: torch.Tensor, seq_lens: torch.Tensor) -> None:
    """move_tokens of checked arguments on the current device."""
    h, nb, steps, dev, kp, vp = lists
    layers, b, _, budget = keep.shape
    rc = _tree.lib().ls_move_tokens(
        kp, vp, layers, steps, nb, block_tables.data_ptr(), block_tables.stride(0),
        block_tables.shape[1], seq_lens.data_ptr(), keep.data_ptr(), b, h, budget, HEAD_DIM, PAGE,
        _lib.stream_of(dev))
    _lib.check(rc, "ls_move_tokens")


def evict_tokens(sums: torch.Tensor, k_pools: Sequence[torch.Tensor],
                 v_pools: Sequence[torch.Tensor], block_tables: torch.Tensor,
                 seq_lens: torch.Tensor, budget: int, sinks: int = 4,
                 recent: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """select_tokens() of sums [L, B, H, T], one layer a pool, and move_tokens() of what it
    keeps: every sequence then has min(seq_lens[b], budget) tokens.  Returns (keep,
    kept): the positions that are rows 0, 1, ... now, and their sums (sums itself is
    left as it is: the caller stores `kept` where the next steps add)."""
    layers = len(k_pools)
    if sums.dim() != 4 or sums.shape[0] != layers or layers != len(v_pools):
        raise ValueError(f"sums must be [{layers}, B, H, T] for {layers} K and {len(v_pools)} V "
                         f"pools, got {tuple(sums.shape)}")
    if not layers:
        return select_tokens(sums, seq_lens, budget, sinks, recent)
    b, h, index = sums.shape[1], sums.shape[2], sums.get_device()
    lists = _tree.pool_lists(k_pools, v_pools)              # (before anything is launched)
    if lists[0] != h:
        raise ValueError(f"sums of {h} heads for pools {tuple(k_pools[0].shape)}")
    width = _tree.tables(block_tables, seq_lens, b, index)
    if k_pools[0].get_device() != index:
        raise ValueError("sums must be on the pools' device")
    _lib.stream_of(sums.device)
    if index != _serving.current_device():
        with torch.cuda.device(sums.device):
            return evict_tokens(sums, k_pools, v_pools, block_tables, seq_lens, budget, sinks,
                                recent)
    keep, kept = select_tokens(sums, seq_lens, budget, sinks, recent)
    if b and width:
        _move(keep, lists, block_tables, seq_lens)
    return keep, kept
