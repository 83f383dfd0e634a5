"""Attention of a tree of drafted tokens over the fp16 paged cache, on HIP kernels.

Speculative decoding checks several drafted continuations of a sequence in one
pass: the drafts form a tree, whose nodes' K and V are written behind the
sequence's (``PagedKVCache.advance(N)``), and every node sees the context, its
ancestors and itself:

    masks, depths = tree_masks(parents)            # once a tree
    out = tree_attention(q, k_pool, v_pool, tables, lens, masks)
    path, lengths, nxt = accept_tokens(tokens, parents, choices, k_pools, v_pools,
                                       tables, lens)

Node 0 is the root: the last token that was chosen, whose K and V are not in the
cache yet.  A node's mask is a row of 64-bit words, bit j % 64 of word j // 64
node j; no masks at all is a chain (several tokens of one continuation).
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from latentserve_amd import _lib, _serving, _tree

HEAD_DIM, PAGE, MAX_NREP, MAX_NODES = _tree.HEAD_DIM, _tree.PAGE, _tree.MAX_NREP, _tree.MAX_NODES
_SCALE = 1.0 / math.sqrt(HEAD_DIM)


class AcceptedTokens(NamedTuple):
    path: torch.Tensor                      # [B, N] int32 nodes in order, -1 behind the last
    lengths: torch.Tensor                   # [B] int32
    next_tokens: torch.Tensor               # [B] int64


def mask_words(nodes: int) -> int:
    return (nodes + 63) // 64


def tree_masks(parents: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """parents [B, N] int32 -> (masks [B, N, words] int64: each node's ancestors and
    itself, depths [B, N] int32: 0 for a node without parent).  A parent comes
    before its children; any other number, like -1, is none.  N is 1..256."""
    if parents.dtype is not torch.int32 or parents.dim() != 2 or not parents.is_contiguous():
        raise ValueError(f"parents must be contiguous int32 [B, N], got {parents.dtype} "
                         f"{tuple(parents.shape)}")
    b, n = parents.shape
    if not 1 <= n <= MAX_NODES:
        raise ValueError(f"a tree has 1..{MAX_NODES} nodes, got {n}")
    dev = parents.device
    stream = _lib.stream_of(dev)
    if dev.index != _serving.current_device():
        with torch.cuda.device(dev):
            return tree_masks(parents)
    masks = torch.empty(b, n, mask_words(n), dtype=torch.int64, device=dev)
    depths = torch.empty(b, n, dtype=torch.int32, device=dev)
    rc = _tree.lib().ls_tree_masks(parents.data_ptr(), masks.data_ptr(), depths.data_ptr(), b, n,
                                   stream)
    _lib.check(rc, "ls_tree_masks")
    return masks, depths


def tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   block_tables: torch.Tensor, seq_lens: torch.Tensor,
                   masks: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                   max_seq_len: Optional[int] = None, softmax_scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None,
                   lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's last N tokens: q [B, N, H, n_rep, 128] fp16 (any
    strides of whole 16 bytes), N 1..256, n_rep 1..16 -> a new tensor of its shape,
    or `out`.

    seq_lens [B] int32 counts the N tokens, whose K and V are in the pools.  Token i
    sees all tokens before the N and, of them, the ones that masks [B, N, words]
    int64 names (None: 0..i).  counts [B] int32 (None: N): a sequence's nodes from
    its count on do not exist: nobody sees them and they give zeros.  A sequence of
    fewer than N tokens is all tree, of so many nodes.

    lse [B, N, H, n_rep] fp32, contiguous, takes the rows' log-sum-exp (natural).  A
    row that sees nothing gives zeros, and -inf there.  K and V that a row does
    not see change nothing, whatever they hold.

    max_seq_len: the longest sequence expected (a graph's bucket); it only sizes the
    launch, a longer one is attended whole.  Blocks outside the pool are skipped.
    out may not overlap q, nor its rows each other.  Each call has its own scratch, so
    calls may run at once on several streams and from several graphs.  The result of a
    call repeats bit for bit."""
    h, nb, steps = _tree.two_pools(k_pool, v_pool)
    shape, dev, index = q.shape, q.device, q.get_device()
    if len(shape) != 5 or shape[2] != h or shape[4] != HEAD_DIM \
            or not 1 <= shape[1] <= MAX_NODES or not 1 <= shape[3] <= MAX_NREP:
        raise ValueError(f"q must be [B, N 1..{MAX_NODES}, {h}, n_rep 1..{MAX_NREP}, {HEAD_DIM}], "
                         f"got {tuple(shape)}")
    if index != k_pool.get_device():
        raise ValueError("q must be on the pools' device")
    b, n, _, n_rep, _ = shape
    width = _tree.tables(block_tables, seq_lens, b, index)
    mp = cp = lp = None
    if masks is not None:
        mp = _tree.whole("masks", masks, torch.int64, (b, n, mask_words(n)), index)
    if counts is not None:
        cp = _tree.whole("counts", counts, torch.int32, (b,), index)
    if lse is not None:
        lp = _tree.whole("lse", lse, torch.float32, (b, n, h, n_rep), index)
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
            return tree_attention(q, k_pool, v_pool, block_tables, seq_lens, masks, counts,
                                  max_seq_len, softmax_scale, out, lse)
    if b == 0 or width == 0:
        if lse is not None:
            lse.fill_(-math.inf)
        return out.zero_()
    bound = _tree.bound_of(max_seq_len, width)
    nbytes = _tree.workspace_bytes("ls_tree_attention_workspace_bytes", b, h, n, n_rep, width, bound)
    work, _ = _serving.scratch(dev, stream, nbytes, 0)
    rc = _tree.lib().ls_tree_attention(
        q.data_ptr(), qs, k_pool.data_ptr(), v_pool.data_ptr(), steps, nb, block_tables.data_ptr(),
        block_tables.stride(0), width, seq_lens.data_ptr(), mp, cp, out.data_ptr(), os, lp,
        work.data_ptr(), nbytes, b, h, n, n_rep, HEAD_DIM, PAGE, bound,
        _SCALE if softmax_scale is None else float(softmax_scale), stream)
    _lib.check(rc, "ls_tree_attention")
    return out


def accept_tokens(tokens: torch.Tensor, parents: torch.Tensor, choices: torch.Tensor,
                  k_pools: Sequence[torch.Tensor], v_pools: Sequence[torch.Tensor],
                  block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  counts: Optional[torch.Tensor] = None) -> AcceptedTokens:
    """The drafted tokens that the model's own choices confirm, and their K and V moved
    together behind the context.

    tokens and choices [B, N] int64: the nodes' tokens, and what the model chose
    after each; parents [B, N] int32 and counts as in tree_masks() and
    tree_attention().  The path starts at node 0 and goes on with the first child
    whose token is its parent's choice; next_tokens is the last one's choice (what
    to feed next: its K and V are not in the cache).  A sequence without nodes has an
    empty path and -1.

    In every layer's pools ([nb, 16, H, 128] fp16, all alike) the path's rows, of the
    sequence's last N tokens (seq_lens [B], which counts them), become the first of
    those: the sequence then is its context and lengths[b] tokens.  What lies behind
    is left over.  A node's place never moves up, so no row is lost.

    The tables of different sequences name different blocks where nodes lie (the
    cache's advance() sees to that)."""
    if tokens.dim() != 2 or not 1 <= tokens.shape[1] <= MAX_NODES:
        raise ValueError(f"tokens must be [B, N 1..{MAX_NODES}], got {tuple(tokens.shape)}")
    if not k_pools:
        raise ValueError("accept_tokens moves the rows of one layer at least")
    b, n = tokens.shape
    h, nb, steps, dev, kp, vp = _tree.pool_lists(k_pools, v_pools)
    index = k_pools[0].get_device()
    tp = _tree.whole("tokens", tokens, torch.int64, (b, n), index)
    pp = _tree.whole("parents", parents, torch.int32, (b, n), index)
    cp = _tree.whole("choices", choices, torch.int64, (b, n), index)
    np_ = None if counts is None else _tree.whole("counts", counts, torch.int32, (b,), index)
    width = _tree.tables(block_tables, seq_lens, b, index)
    stream = _lib.stream_of(dev)
    if index != _serving.current_device():
        with torch.cuda.device(dev):
            return accept_tokens(tokens, parents, choices, k_pools, v_pools, block_tables, seq_lens,
                                 counts)
    path = torch.empty(b, n, dtype=torch.int32, device=dev)
    lengths = torch.empty(b, dtype=torch.int32, device=dev)
    nxt = torch.empty(b, dtype=torch.int64, device=dev)
    if b:
        if width == 0:
            raise ValueError("block tables without pages")
        rc = _tree.lib().ls_accept_tokens(
            tp, pp, cp, np_, path.data_ptr(), lengths.data_ptr(), nxt.data_ptr(), kp, vp,
            len(k_pools), steps, nb, block_tables.data_ptr(), block_tables.stride(0), width,
            seq_lens.data_ptr(), b, h, n, HEAD_DIM, PAGE, stream)
        _lib.check(rc, "ls_accept_tokens")
    return AcceptedTokens(path, lengths, nxt)
