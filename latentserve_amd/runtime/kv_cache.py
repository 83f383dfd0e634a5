"""Paged KV cache bookkeeping for the HIP decode path.

The reference's cache layer (cache/block_allocator.py: BlockAllocator,
BlockTable, OutOfBlocks; cache/paged_cache.py: PagedKVCache) fixes what
the kernels read: per-layer pools ``[num_blocks, 16, H_kv, D]``, a block
table per sequence whose token p lives at flat slot ``blocks[p // 16] * 16
+ p % 16``, blocks handed out lowest id first and reused most recently
freed first.  Those rules are kept; the machinery is this build's own:

* ``StepInputs`` holds every per-step kernel input at a fixed device
  address (a captured graph reads them by pointer): the block-table rows
  at the cache's capacity width, the lengths, the decode token's write
  slot, and for the INT8 cache the residual row and index.  The per-step
  vectors live in one device buffer filled by ONE host-to-device copy from
  a double-buffered pinned staging area; a table row is uploaded only
  where it changed, and a row that only grew uploads just its new tail.
* The allocator keeps a reference count per block id in a flat list and
  the free ids on a stack.

Host-side Python, like the reference's: a decode step's bookkeeping is a
few list operations and one small copy.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Dict, Iterable, List, Optional, Sequence

import numpy as np
import torch


class OutOfBlocks(RuntimeError):
    """The pool cannot hold the requested blocks (cache/block_allocator.py:
    31-38): a scheduler's signal to wait or evict, not a crash."""


class BlockAllocator:
    """A fixed pool of equal blocks (cache/block_allocator.py:41-132).

    A fresh pool hands out 0, 1, 2, ...; a freed block is the next one
    handed out (most recently freed first).  Blocks are reference counted
    so a shared prefix can be held by several sequences.

    Three optional hooks let a prefix cache lend the pool the blocks only it
    still holds (cache/block_allocator.py:60-67, 100-103, 131-142):
    ``reclaimable()`` counts them (admission sees them as available),
    ``reclaimer(n)`` gives up to n of them back when an allocation comes up
    short, and ``on_ref_change(block, old, new)`` reports every count change.
    """

    def __init__(self, num_blocks: int, block_size: int):
        if num_blocks < 1 or block_size < 1:
            raise ValueError(f"a pool needs at least one block of at least one token "
                             f"(got {num_blocks} blocks of {block_size})")
        self.num_blocks = int(num_blocks)
        self.block_size = int(block_size)
        self._refs: List[int] = [0] * self.num_blocks
        self._stack: List[int] = []
        self.peak_used = 0
        self.alloc_calls = 0
        self.free_calls = 0
        self.reclaimer: Optional[Callable[[int], object]] = None
        self.reclaimable: Optional[Callable[[], int]] = None
        self.on_ref_change: Optional[Callable[[int, int, int], None]] = None
        # told of compact()'s moves, {old block: new block}, once they are made
        self.on_move: Optional[Callable[[Dict[int, int]], None]] = None
        self.reset()

    def reset(self) -> None:
        """Every block free again and the counters at zero: the pool as new."""
        self._refs = [0] * self.num_blocks
        self._stack = list(range(self.num_blocks - 1, -1, -1))   # top = lowest id
        self.peak_used = self.alloc_calls = self.free_calls = 0

    def stats(self) -> dict:
        """The pool's occupancy and traffic, under the reference's keys
        (cache/block_allocator.py:152-161)."""
        return {"num_blocks": self.num_blocks, "block_size": self.block_size,
                "blocks_used": self.num_used, "blocks_free": self.num_free,
                "block_utilization": self.utilization, "peak_blocks_used": self.peak_used,
                "alloc_calls": self.alloc_calls, "free_calls": self.free_calls}

    @property
    def num_free(self) -> int:
        return len(self._stack)

    @property
    def num_used(self) -> int:
        return self.num_blocks - len(self._stack)

    @property
    def utilization(self) -> float:
        return self.num_used / self.num_blocks

    def blocks_for_tokens(self, num_tokens: int) -> int:
        return -(-int(num_tokens) // self.block_size)

    @property
    def num_available(self) -> int:
        """What an allocation can get: free blocks, and blocks a prefix
        cache holds alone."""
        return len(self._stack) + (self.reclaimable() if self.reclaimable else 0)

    def ensure(self, count: int) -> None:
        """`count` blocks free, reclaimed where it takes that; else OutOfBlocks."""
        if count > len(self._stack) and self.reclaimer is not None:
            self.reclaimer(count - len(self._stack))
        if count > len(self._stack):
            raise OutOfBlocks(f"cannot allocate {count} blocks: only {len(self._stack)} of "
                              f"{self.num_blocks} are free")

    def allocate(self, count: int) -> List[int]:
        count = int(count)
        self.ensure(count)
        taken = self._stack[len(self._stack) - count:][::-1]
        del self._stack[len(self._stack) - count:]
        self.alloc_calls += 1
        for b in taken:
            self._refs[b] = 1
        self.peak_used = max(self.peak_used, self.num_used)
        return taken

    def incref(self, blocks: Iterable[int]) -> None:
        for b in blocks:
            if not 0 <= b < self.num_blocks or self._refs[b] == 0:
                raise ValueError(f"block {b} is free; only allocated blocks can be shared")
            self._refs[b] += 1
            if self.on_ref_change is not None:
                self.on_ref_change(b, self._refs[b] - 1, self._refs[b])

    def free(self, blocks: Iterable[int]) -> None:
        """Drop one reference to each block; a block whose count reaches
        zero goes back on the stack."""
        self.free_calls += 1
        for b in blocks:
            if not 0 <= b < self.num_blocks or self._refs[b] == 0:
                raise ValueError(f"block {b} is already free")
            self._refs[b] -= 1
            if self._refs[b] == 0:
                self._stack.append(b)
            if self.on_ref_change is not None:
                self.on_ref_change(b, self._refs[b] + 1, self._refs[b])

    def compacting_moves(self) -> Dict[int, int]:
        """{old: new}, ascending: the held blocks past the pool's first num_used go to
        its free ones below, after which the held blocks are 0 .. num_used - 1."""
        n = self.num_used
        low = [b for b in range(n) if self._refs[b] == 0]
        return dict(zip((b for b in range(n, self.num_blocks) if self._refs[b]), low))

    def move(self, moves: Dict[int, int]) -> None:
        """Renumber held blocks (their contents have been copied): counts move along,
        the free blocks are handed out lowest first again."""
        for old, new in moves.items():
            self._refs[new], self._refs[old] = self._refs[old], 0
        self._stack = [b for b in range(self.num_blocks - 1, -1, -1) if self._refs[b] == 0]
        if self.on_move is not None:
            self.on_move(moves)

    def ref_count(self, block: int) -> int:
        return self._refs[block]

    refcount = ref_count


class BlockTable:
    """One sequence's pages (cache/block_allocator.py:165-229).

    ``blocks``: physical ids in logical order; ``length``: tokens written;
    ``version``: bumped whenever ``blocks`` changes (a new page, a free), so
    a mirror of the table knows to refresh.
    """

    def __init__(self, allocator: BlockAllocator):
        self.allocator = allocator
        self.blocks: List[int] = []
        self.length = 0
        self.version = 0
        # bumped when the block list is replaced rather than extended: a
        # mirror that saw an older lineage re-uploads the whole row
        self.lineage = 0
        # tokens that were evicted: rows are no longer the tokens of their numbers, and the
        # next token's position is length + dropped
        self.dropped = 0
        # the first row from which on all heads hold the same tokens: what lies before it was
        # chosen head by head, so a sequence can be shortened to it, or to nothing
        self.common = 0

    @property
    def capacity(self) -> int:
        """Token slots of the table's pages."""
        return len(self.blocks) * self.allocator.block_size

    @property
    def wasted_slots(self) -> int:
        """Slots of the last page past the tokens written (internal
        fragmentation, under one page a sequence)."""
        return self.capacity - self.length

    def reserve(self, num_tokens: int) -> None:
        """Pages for length + num_tokens tokens, allocated as needed; the
        length is unchanged (cache/block_allocator.py:198-208)."""
        need = self.allocator.blocks_for_tokens(self.length + num_tokens) - len(self.blocks)
        if need > 0:
            self.blocks.extend(self.allocator.allocate(need))
            self.version += 1

    def append(self, num_tokens: int) -> None:
        """Make room for num_tokens more tokens (new pages as needed)."""
        self.reserve(num_tokens)
        self.length += num_tokens

    def slot(self, position: int) -> int:
        if not 0 <= position < self.length:
            raise IndexError(f"position {position} is outside the sequence (length "
                             f"{self.length})")
        page, off = divmod(position, self.allocator.block_size)
        return self.blocks[page] * self.allocator.block_size + off

    def slots(self, start: int = 0, end: Optional[int] = None) -> List[int]:
        end = self.length if end is None else end
        return [self.slot(p) for p in range(start, end)]

    def free(self) -> None:
        self.allocator.free(self.blocks)
        self.blocks = []
        self.length = 0
        self.version += 1
        self.lineage += 1
        self.dropped = self.common = 0


@dataclass
class KVCacheSpec:
    """Geometry of a cache (the fields of the reference's cache/kv_cache.py
    KVCacheSpec that a paged cache reads)."""

    num_layers: int
    num_kv_heads: int
    head_dim: int
    max_batch_size: int
    max_seq_len: int
    dtype: torch.dtype = torch.float16
    device: str = "cuda"


class StepInputs:
    """Per-step kernel inputs at fixed device addresses.

    ``tables`` [max_batch, capacity_pages] int32, and five vectors of
    max_batch entries carved from one device buffer: ``write_slot`` int64
    (the decode token's flat slot), ``res_index`` int64 (its row in the
    flattened INT8 residual), ``lens`` int32, ``res_row`` int32 (each
    sequence's residual row) and ``slot`` int32 (its slot, where weight sums
    are kept).  ``publish`` writes the step's values into a
    pinned staging area and issues asynchronous copies: the changed table
    entries, then the whole vector buffer in one copy.  Two staging areas
    alternate; one is refilled only after the copies that last read it
    have run, so the host never waits for the step before.
    """

    _FIELDS = (("write_slot", np.int64), ("res_index", np.int64),
               ("lens", np.int32), ("res_row", np.int32), ("slot", np.int32))

    def __init__(self, max_batch: int, capacity_pages: int, block_size: int, device):
        self.max_batch = mb = int(max_batch)
        self.capacity_pages = cap = max(1, int(capacity_pages))
        self.block_size = int(block_size)
        self.device = torch.device(device)
        self.tables = torch.zeros((mb, cap), dtype=torch.int32, device=self.device)
        offs, pos = {}, 0
        for name, dt in self._FIELDS:
            offs[name] = (pos, pos + mb * np.dtype(dt).itemsize)
            pos = offs[name][1]
        self._dev = torch.zeros(pos, dtype=torch.uint8, device=self.device)
        self.vec = {name: self._dev[a:b].view(_TORCH[dt])
                    for (name, dt), (a, b) in zip(self._FIELDS, offs.values())}
        # the values of every field as last published (host copy)
        self._cur = np.zeros(pos, dtype=np.uint8)
        self._cur_views = {name: self._cur[a:b].view(dt)
                           for (name, dt), (a, b) in zip(self._FIELDS, offs.values())}
        self._async = self.device.type == "cuda"
        self._stage = []
        for _ in range(2 if self._async else 1):
            vec = torch.zeros(pos, dtype=torch.uint8, pin_memory=self._async)
            tab = torch.zeros((mb, cap), dtype=torch.int32, pin_memory=self._async)
            self._stage.append((vec, tab, torch.cuda.Event() if self._async else None))
        self._turn = 0
        # per table row: (sequence slot, its lineage, entries uploaded)
        self._row_state: List[Optional[tuple]] = [None] * mb

    def forget_rows(self) -> None:
        self._row_state = [None] * self.max_batch

    def publish(self, seqs: Sequence[int], tables: Sequence[BlockTable],
                **values: Sequence[int]) -> None:
        """Row r of the device table mirrors tables[seqs[r]].blocks; each
        vector given is set for rows 0..len-1 (vectors not given keep their
        last published values)."""
        if self._async:
            self._turn ^= 1
        vec, tab, ev = self._stage[self._turn]
        if ev is not None:
            ev.synchronize()                    # the copies that last read this area ran
        tab_np = tab.numpy()
        for row, s in enumerate(seqs):
            t = tables[s]
            n = len(t.blocks)
            if n > self.capacity_pages:
                raise RuntimeError(f"the sequence in slot {s} holds {n} pages; the cache was "
                                   f"sized for {self.capacity_pages}")
            st = self._row_state[row]
            first = st[2] if st is not None and st[0] == s and st[1] == t.lineage \
                and st[2] <= n else 0
            if first < n:
                tab_np[row, first:n] = t.blocks[first:n]
                self.tables[row, first:n].copy_(tab[row, first:n], non_blocking=self._async)
            self._row_state[row] = (s, t.lineage, n)
        for name, vals in values.items():
            self._cur_views[name][:len(vals)] = vals
        vec.numpy()[:] = self._cur
        self._dev.copy_(vec, non_blocking=self._async)
        if ev is not None:
            ev.record()


NO_SPARSE_SUMS = "a sparse step does not see all weights that the cache is to sum"

_TORCH = {np.int64: torch.int64, np.int32: torch.int32}


class _PagedBase:
    """Bookkeeping shared by the fp16 and INT8 paged caches: allocator,
    per-slot tables, the active set, and the kernel inputs."""

    def __init__(self, spec: KVCacheSpec, block_size: int, num_blocks: Optional[int]):
        if block_size != 16:
            raise ValueError(f"the HIP kernels read 16-token pages, not {block_size}")
        self.spec = spec
        self.block_size = block_size
        self.device = torch.device(spec.device)
        self.capacity_pages = -(-spec.max_seq_len // block_size)
        self.num_blocks = num_blocks or self.capacity_pages * spec.max_batch_size
        self.allocator = BlockAllocator(self.num_blocks, block_size)
        self.tables = [BlockTable(self.allocator) for _ in range(spec.max_batch_size)]
        self.inputs = StepInputs(spec.max_batch_size, self.capacity_pages, block_size,
                                 self.device)
        self._active: List[int] = list(range(spec.max_batch_size))
        self._batch = 0                       # rows published by the last advance()
        self._rows: List[int] = []            # and whose they are
        self._chunk_slots: Optional[torch.Tensor] = None    # multi-token write slots
        # Positions that the model has (None: no bound but the cache's capacity).  Sequences
        # that lost tokens get past the capacity.
        self.max_positions: Optional[int] = None
        # Whether the model's steps are sparse (its set_sparse()): they see a part of the tokens.
        self.sparse = False
        # When set (a graph runner's bucket), sparse selection is sized for it.
        self.sparse_context_hint: Optional[int] = None

    # ---- the active set ---------------------------------------------------
    @property
    def seq_lens(self) -> List[int]:
        return [self.tables[s].length for s in self._active]

    @property
    def seq_positions(self) -> List[int]:
        """The active sequences' next positions: tokens held and tokens evicted."""
        return [self.tables[s].length + self.tables[s].dropped for s in self._active]

    @property
    def max_len(self) -> int:
        return max((self.tables[s].length for s in self._active), default=0)

    @property
    def active_slots(self) -> List[int]:
        return list(self._active)

    def set_active(self, slots: Sequence[int]) -> None:
        self._active = list(slots)

    def can_admit(self, num_tokens: int) -> bool:
        """Whether a prompt of num_tokens fits now (blocks a prefix cache
        holds alone count: an allocation reclaims them)."""
        return self.allocator.blocks_for_tokens(num_tokens) <= self.allocator.num_available

    def free_sequence(self, index: int) -> None:
        self.tables[index].free()

    # ---- prefix sharing ---------------------------------------------------
    def attach_prefix(self, index: int, blocks: Sequence[int], num_tokens: int) -> None:
        """Start the empty slot `index` on `blocks`, whole pages already
        written by another sequence with the same first num_tokens tokens
        (cache/paged_cache.py:199-217).  The slot takes a reference to each;
        a step that would write a page that others hold too (a rewound or forked
        sequence's) gives its sequence a copy first (_make_room())."""
        t = self.tables[index]
        if t.length or t.blocks:
            raise ValueError(f"slot {index} already holds a sequence")
        if num_tokens != len(blocks) * self.block_size:
            raise ValueError(f"a shared prefix is whole pages: {len(blocks)} pages hold "
                             f"{len(blocks) * self.block_size} tokens, not {num_tokens}")
        self.allocator.incref(blocks)
        t.blocks = list(blocks)
        t.length = int(num_tokens)
        t.version += 1
        t.lineage += 1

    def shareable_blocks(self, index: int) -> int:
        """Leading pages of slot `index` whose K/V in the pool is final, so a
        prefix cache may hand them to another sequence (of a sequence that lost
        tokens, none: its pages are not of the prompt's first tokens)."""
        t = self.tables[index]
        return 0 if t.dropped else t.length // self.block_size

    # ---- branching and compaction -------------------------------------------
    def _page_tensors(self) -> List[torch.Tensor]:
        """Every tensor indexed by block, all layers'."""
        raise NotImplementedError

    def _copy_rows(self, tensors: Sequence[torch.Tensor], src: Sequence[int],
                   dst: Sequence[int]) -> None:
        if not src:
            return
        if self.device.type == "cuda":
            from latentserve_amd.kernels.hip import page_copy as pc
            pc.copy_pages(tensors, src, dst)
        else:
            for t in tensors:
                t[list(dst)] = t[list(src)]

    def fork(self, index: int, children: Sequence[int]) -> None:
        """Branch the sequence in slot `index` into the empty slots `children`: each
        holds the same tokens, on the same pages, and grows its own way from
        there.  Nothing is copied now: a page that several sequences hold is
        copied when one of them is about to write it (advance()).  Between
        steps only: the tokens of the last advance() must have been written
        (the caller's to see to: a replayed graph's writes pass the cache by)."""
        children = list(children)
        for s in [index] + children:
            if not 0 <= s < len(self.tables):
                raise ValueError(f"slot {s} is not one of {len(self.tables)}")
        t = self.tables[index]
        if len(set(children)) != len(children):
            raise ValueError(f"slots {children}: a child is named twice")
        for c in children:
            if c == index or self.tables[c].length or self.tables[c].blocks:
                raise ValueError(f"slot {c} already holds a sequence")
        pages = t.blocks[:self.allocator.blocks_for_tokens(t.length)]
        for c in children:
            child = self.tables[c]
            self.allocator.incref(pages)
            child.blocks = list(pages)
            child.length = t.length
            child.dropped, child.common = t.dropped, t.common
            child.version += 1
            child.lineage += 1

    def _make_room(self, seqs: Sequence[int], n: int) -> None:
        """Pages for n more tokens of each sequence, lengths unchanged; and of the pages
        they go to, those that other sequences (or a prefix cache) hold too are
        replaced by pages of their own, with the tokens they keep.  All or
        nothing: where the pool has not the blocks for all of it (OutOfBlocks),
        or a sequence would outgrow the cache, nothing has changed."""
        bs = self.block_size
        spans, grown = [], 0
        for s in seqs:
            t = self.tables[s]
            if t.dropped and self.max_positions is not None \
                    and t.length + t.dropped + n > self.max_positions:
                raise RuntimeError(f"the sequence in slot {s} would reach position "
                                   f"{t.length + t.dropped + n - 1}; the model was given "
                                   f"{self.max_positions}")
            first, have, end = t.length // bs, len(t.blocks), -(-(t.length + n) // bs)
            if end > have:
                if end > self.capacity_pages:
                    raise RuntimeError(f"the sequence in slot {s} would hold {end} pages; the "
                                       f"cache was sized for {self.capacity_pages}")
                grown += end - have
            spans.append((t, first, min(have, end), first + (t.length % bs > 0)))
        self._own_pages(spans, grown)
        if grown:
            for s in seqs:
                self.tables[s].reserve(n)

    def _own_pages(self, spans, grown: int = 0) -> None:
        """Of each (table, first, end, kept), the pages first .. end - 1 that others hold too
        replaced by pages of its own, with what the ones before `kept` hold.  All or
        nothing, as is room for `grown` blocks more."""
        refs = self.allocator.ref_count
        todo, left = [], {}
        for t, first, end, kept in spans:
            for page in range(first, end):
                blk = t.blocks[page]
                count = left.get(blk, refs(blk))
                if count > 1:
                    left[blk] = count - 1              # the last to write keeps the page
                    todo.append((t, page, blk, page < kept))
        if grown or todo:
            self.allocator.ensure(grown + len(todo))
        if todo:
            fresh = self.allocator.allocate(len(todo))
            kept = [(blk, new) for (_, _, blk, keeps), new in zip(todo, fresh) if keeps]
            self._copy_rows(self._page_tensors(), [a for a, _ in kept], [b for _, b in kept])
            for (t, page, blk, _), new in zip(todo, fresh):
                t.blocks[page] = new
                t.version += 1
                t.lineage += 1
            self.allocator.free([blk for _, _, blk, _ in todo])

    def compact(self) -> Dict[int, int]:
        """Move the held pages to the pool's lowest blocks, so that they are blocks
        0 .. num_used - 1 (one slice a tensor to save, send or trim), and
        renumber them in the tables and the prefix cache.  Returns the moves, {old
        block: new block}, for holders the cache does not know.  Between
        steps only, as fork(); captured graphs stay valid."""
        moves = self.allocator.compacting_moves()
        if moves:
            self._copy_rows(self._page_tensors(), list(moves), list(moves.values()))
            for t in self.tables:
                if any(b in moves for b in t.blocks):
                    t.blocks = [moves.get(b, b) for b in t.blocks]
                    t.version += 1
                    t.lineage += 1
            self.allocator.move(moves)
            if self._batch:
                self._publish(0, [self.tables[s].length for s in self._active])
        return moves

    def _shorten(self, length: int, seqs: Sequence[int]) -> None:
        for s in seqs:
            t = self.tables[s]
            if not 0 <= length <= t.length:
                raise ValueError(f"slot {s} holds {t.length} tokens; cannot rewind it to "
                                 f"{length}")
            if 0 < length < t.common:
                raise ValueError(f"slot {s} holds different tokens in each head before row "
                                 f"{t.common}, where others were evicted; cannot rewind it to "
                                 f"{length}")
        for s in seqs:
            t = self.tables[s]
            t.length = length
            if length == 0:                            # (nothing is held: a new sequence)
                t.dropped = t.common = 0

    def reset(self) -> None:
        """Forget every sequence; storage (and every address a graph holds)
        is kept."""
        for t in self.tables:
            if t.blocks:
                t.free()
        self.allocator.reset()
        self._active = list(range(self.spec.max_batch_size))
        self._batch, self._rows = 0, []
        self._chunk_slots = None
        self.inputs.forget_rows()

    # ---- per-step inputs --------------------------------------------------
    def _room_for_step(self, n: int, batch_size, slots) -> None:
        """The sequences that a step extends become the active ones, with room for n more
        tokens each; where there is none, nothing has changed."""
        seqs = list(slots) if slots is not None else \
            self._active if batch_size is None else list(range(batch_size))
        if len(set(seqs)) != len(seqs):
            raise ValueError(f"slots {seqs}: a sequence is named twice")
        if n:                              # (a step of none writes no page: it shares on)
            self._make_room(seqs, n)
        self._active = seqs

    def _grow(self, n: int) -> List[int]:
        """Extend the active sequences by n tokens, which there is room for; returns
        their old lengths."""
        starts = [self.tables[s].length for s in self._active]
        for s in self._active:
            self.tables[s].length += n
        return starts

    def _publish(self, n: int, starts: List[int], extra: Optional[dict] = None) -> None:
        seqs = self._active
        vals = {"lens": [self.tables[s].length for s in seqs]}
        if n == 1:
            vals["write_slot"] = [self.tables[s].slot(p) for s, p in zip(seqs, starts)]
            self._chunk_slots = None
        else:
            self._chunk_slots = torch.from_numpy(
                self._token_slots(seqs, starts, n)).to(self.device)
        vals.update(extra or {})
        self.inputs.publish(seqs, self.tables, **vals)
        self._batch, self._rows = len(seqs), list(seqs)

    def _token_slots(self, seqs: Sequence[int], starts: Sequence[int], n: int) -> np.ndarray:
        """[len(seqs), n] int64 flat slots of tokens start .. start + n - 1 of
        each sequence, from its pages (a page at a time: BlockTable.slot
        a token was 0.8 ms of a pass that writes 4 prompts of 2048 tokens)."""
        bs = self.block_size
        out = np.empty((len(seqs), n), dtype=np.int64)
        if n:
            offs = np.arange(bs, dtype=np.int64)
            for row, (s, p) in enumerate(zip(seqs, starts)):
                first = p // bs
                blocks = np.asarray(self.tables[s].blocks[first:(p + n - 1) // bs + 1], np.int64)
                p -= first * bs
                out[row] = (blocks[:, None] * bs + offs).reshape(-1)[p:p + n]
        return out

    def _need(self, b: Optional[int]) -> int:
        if self._batch == 0:
            raise RuntimeError("advance() the cache before asking for kernel inputs")
        b = self._batch if b is None else int(b)
        if b > self._batch:
            raise RuntimeError(f"{b} rows asked for, the last advance() published "
                               f"{self._batch}")
        return b

    def block_tables_tensor(self, batch_size: Optional[int] = None) -> torch.Tensor:
        """[B, capacity_pages] int32 rows of the active sequences (fixed address)."""
        return self.inputs.tables[:self._need(batch_size)]

    def seq_lens_tensor(self, batch_size: Optional[int] = None) -> torch.Tensor:
        return self.inputs.vec["lens"][:self._need(batch_size)]

    def write_slots(self, batch_size: int) -> torch.Tensor:
        """[B] int64 flat slot of each active sequence's decode token (after
        an advance(1)), at a fixed address."""
        if self._chunk_slots is not None:
            raise RuntimeError("the last advance() reserved several tokens; write_slots() "
                               "names the single decode token of an advance(1)")
        return self.inputs.vec["write_slot"][:self._need(batch_size)]

    def _slots_for_write(self, b: int, n: int) -> torch.Tensor:
        """[b, n] flat slots the last advance() reserved."""
        if n == 1 and self._chunk_slots is None:
            return self.inputs.vec["write_slot"][:self._need(b)].view(b, 1)
        if self._chunk_slots is None or self._chunk_slots.shape != (b, n):
            raise RuntimeError(f"advance({n}) for {b} sequences must precede this write")
        return self._chunk_slots


class PagedKVCache(_PagedBase):
    """fp16 paged KV storage (cache/paged_cache.py:63-506), decode side."""

    def __init__(self, spec: KVCacheSpec, block_size: int = 16, num_blocks: Optional[int] = None):
        super().__init__(spec, block_size, num_blocks)
        shape = (self.num_blocks, block_size, spec.num_kv_heads, spec.head_dim)
        self.k_pool = [torch.zeros(shape, dtype=spec.dtype, device=self.device)
                       for _ in range(spec.num_layers)]
        self.v_pool = [torch.zeros(shape, dtype=spec.dtype, device=self.device)
                       for _ in range(spec.num_layers)]
        self.kmin: Optional[List[torch.Tensor]] = None
        self.kmax: Optional[List[torch.Tensor]] = None
        # [layers, slots, heads, tokens] fp32: see enable_weight_sums()
        self.weight_sums: Optional[torch.Tensor] = None

    def _page_tensors(self) -> List[torch.Tensor]:
        return self.k_pool + self.v_pool + (self.kmin or []) + (self.kmax or [])

    def advance(self, n: int, batch_size: Optional[int] = None,
                slots: Optional[Sequence[int]] = None) -> None:
        """Reserve n more tokens for each active sequence (paged_cache.py:
        235-271) and publish the step's kernel inputs.  OutOfBlocks leaves
        every sequence, and which are active, as they were."""
        self._room_for_step(n, batch_size, slots)
        if self.weight_sums is not None:
            for s in self._active:
                if not self.tables[s].length:          # (what the slot's last sequence left)
                    self.weight_sums[:, s].zero_()
        self._publish(n, self._grow(n))

    def _publish(self, n: int, starts: List[int], extra: Optional[dict] = None) -> None:
        if self.weight_sums is not None:
            extra = {**(extra or {}), "slot": self._active}
        super()._publish(n, starts, extra)

    def rewind(self, length: int, slots: Optional[Sequence[int]] = None) -> None:
        """Shorten sequences to `length` tokens, keeping their pages
        (paged_cache.py:273-303): growing again lands on the same slots.  A sequence
        that lost tokens can be rewound to nothing, which starts it anew, or to its
        most recent tokens (the `recent` that evict() kept, and later ones): the rows
        before them are different tokens in each head."""
        seqs = self._active if slots is None else list(slots)
        before = [self.tables[s].length for s in seqs]
        self._shorten(length, seqs)
        if self.kmin is not None and length % self.block_size:
            try:
                # (its bounds change: no one else's may)
                self._make_room(list(dict.fromkeys(seqs)), 0)
            except OutOfBlocks:
                for s, n in zip(seqs, before):
                    self.tables[s].length = n
                raise
            for s in seqs:
                self._bound_partial_page(s, length)
        if self.weight_sums is not None:
            for s in seqs:
                self.weight_sums[:, s, :, length:].zero_()
        self._publish(0, [self.tables[s].length for s in self._active])

    def fork(self, index: int, children: Sequence[int]) -> None:
        children = list(children)
        super().fork(index, children)
        if self.weight_sums is not None:
            for c in children:
                self.weight_sums[:, c].copy_(self.weight_sums[:, index])

    def attach_prefix(self, index: int, blocks: Sequence[int], num_tokens: int) -> None:
        super().attach_prefix(index, blocks, num_tokens)
        if self.weight_sums is not None:
            self.weight_sums[:, index].zero_()

    # ---- drafted trees and a bounded cache ----------------------------------
    def accept(self, tokens: torch.Tensor, parents: torch.Tensor, choices: torch.Tensor,
               counts: Optional[torch.Tensor] = None):
        """End a step of drafted trees: the active sequences hold N drafted tokens each
        (advance(N), then a pass that wrote them), and keep the ones that the model's own
        choices confirm, moved together behind their context
        (kernels.hip.tree_attention.accept_tokens, whose arguments and result these
        are).  The lengths that the host keeps follow, so this waits for the
        GPU."""
        from latentserve_amd.kernels.hip import tree_attention as ta

        seqs = self._active
        if seqs != self._rows:
            raise RuntimeError(f"slots {seqs} are active, the last step was of slots {self._rows}: "
                               "accept() ends the step that advance() began")
        if tokens.dim() != 2 or tokens.shape[0] != self._need(None):
            raise ValueError(f"tokens must be [{self._need(None)}, N], got {tuple(tokens.shape)}")
        n = tokens.shape[1]
        for s in seqs:
            if self.tables[s].length - n < self.tables[s].common:
                raise ValueError(f"slot {s} holds {self.tables[s].length} tokens, not {n} drafted "
                                 "ones")
        got = ta.accept_tokens(tokens, parents, choices, self.k_pool, self.v_pool,
                               self.block_tables_tensor(), self.seq_lens_tensor(), counts)
        for s, m in zip(seqs, got.lengths.tolist()):
            t = self.tables[s]
            before = t.length - n
            t.length = before + m
            self._bound_pages(s, before // self.block_size)
        self._publish(0, [self.tables[s].length for s in seqs])
        return got

    def enable_weight_sums(self) -> None:
        """Keep, per layer, slot and KV head, the attention weight that each cached token
        has got so far (the decoder's dense steps add to it), for evict().  A sequence's
        sums follow it through rewind(), fork() and accept(); they start at zero: of
        tokens that were written without such a step (a prompt's chunks, a shared
        prefix), evict() knows nothing but their places."""
        if self.sparse:
            raise ValueError(NO_SPARSE_SUMS)
        if self.weight_sums is None:
            spec = self.spec
            self.weight_sums = torch.zeros(spec.num_layers, spec.max_batch_size, spec.num_kv_heads,
                                           self.capacity_pages * self.block_size,
                                           dtype=torch.float32, device=self.device)
            if self._batch:
                self._publish(0, [self.tables[s].length for s in self._active])

    def sum_rows_tensor(self, batch_size: Optional[int] = None) -> torch.Tensor:
        """[B] int32 slots of the active sequences, their rows of a layer's weight sums
        (fixed address)."""
        return self.inputs.vec["slot"][:self._need(batch_size)]

    def evict(self, budget: int, sinks: int = 4, recent: Optional[int] = None,
              slots: Optional[Sequence[int]] = None) -> List[int]:
        """Bring the active sequences (or `slots`) to at most `budget` tokens each: per
        layer and KV head, the first `sinks`, the last `recent` (default: a quarter of
        the budget) and those with the largest weight sums of the others, moved to
        the front (kernels.hip.cache_eviction.evict_tokens).  Their pages behind go
        back to the pool; pages that others hold are copied first.  Returns the slots
        that lost tokens.  A sequence's length then is no longer its next token's
        position (seq_positions).  Between steps only, as fork(); OutOfBlocks leaves
        every sequence as it was."""
        from latentserve_amd.kernels.hip import cache_eviction as ce

        if self.weight_sums is None:
            raise RuntimeError("enable_weight_sums() before the steps that eviction goes by")
        budget, sinks, recent = ce.budget_of(budget, sinks, recent)
        seqs = list(dict.fromkeys(self._active if slots is None else slots))
        for s in seqs:
            if not 0 <= s < len(self.tables):
                raise ValueError(f"slot {s} is not one of {len(self.tables)}")
        seqs = [s for s in seqs if self.tables[s].length > budget]
        if not seqs:
            return []
        tables = [self.tables[s] for s in seqs]
        pages = -(-budget // self.block_size)
        self._own_pages([(t, 0, pages, pages) for t in tables])
        width = max(len(t.blocks) for t in tables)
        rows = torch.tensor([t.blocks + [0] * (width - len(t.blocks)) for t in tables],
                            dtype=torch.int32).to(self.device)
        lens = torch.tensor([t.length for t in tables], dtype=torch.int32).to(self.device)
        at = torch.tensor(seqs).to(self.device)
        _, kept = ce.evict_tokens(self.weight_sums[:, at], self.k_pool, self.v_pool, rows, lens,
                                  budget, sinks, recent)
        self.weight_sums[:, at] = 0
        self.weight_sums[:, at, :, :budget] = kept
        for s, t in zip(seqs, tables):
            lost = t.length - budget
            t.dropped += lost
            t.common = max(budget - recent, t.common - lost)
            t.length = budget
            self.allocator.free(t.blocks[pages:])
            t.blocks = t.blocks[:pages]
            t.version += 1
            t.lineage += 1
            self._bound_pages(s, 0)
        if self._batch:
            self._publish(0, [self.tables[s].length for s in self._active])
        return seqs

    def write(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, start_pos: int = 0) -> None:
        """Store k, v [B, H_kv, n, D] at the slots the last advance(n) reserved."""
        b, h, n, d = k.shape
        from latentserve_amd.kernels.hip import paged_write as pw

        flat = self._slots_for_write(b, n).reshape(-1)
        k_pool, v_pool = self.k_pool[layer_idx], self.v_pool[layer_idx]
        bounds = None if self.kmin is None else (self.kmin[layer_idx], self.kmax[layer_idx])
        # a chunk's bounds are rebuilt over the pool by the same call
        done = pw.write(k, v, flat, k_pool, v_pool, bounds if n != 1 else None)
        if not done:                # a CPU cache, or rows the kernel's 16-byte loads cannot take
            rows_k = k.transpose(1, 2).reshape(b * n, h, d)
            rows_v = v.transpose(1, 2).reshape(b * n, h, d)
            k_pool.view(-1, h, d).index_copy_(0, flat, rows_k)
            v_pool.view(-1, h, d).index_copy_(0, flat, rows_v)
        if bounds is not None and (n == 1 or not done):
            from latentserve_amd.kernels.hip import paged_sparse as ps
            if n == 1:
                ps.update_bounds(k[:, :, 0], flat, *bounds)
            else:
                ps.rebuild_bounds(k_pool, *bounds)

    def read(self, layer_idx: int, batch_size: int, length: Optional[int] = None):
        """[B, H_kv, L, D] K and V of the active sequences (the gather read,
        paged_cache.py:486-506), on the HIP gather kernel."""
        from latentserve_amd.kernels.hip import paged_gather as pg

        length = self.max_len if length is None else length
        return pg.read(self.k_pool[layer_idx], self.v_pool[layer_idx],
                       self.block_tables_tensor(batch_size), self.seq_lens_tensor(batch_size),
                       length)

    # ---- page bounds for the sparse indexer -------------------------------
    def enable_page_bounds(self) -> None:
        """Per-block per-channel K min / max per layer (paged_cache.py:422-445),
        built from the pools and kept current by every write."""
        if self.kmin is not None:
            return
        nb, _, h, d = self.k_pool[0].shape
        self.kmin = [torch.zeros(nb, h, d, dtype=self.spec.dtype, device=self.device)
                     for _ in self.k_pool]
        self.kmax = [torch.zeros_like(t) for t in self.kmin]
        from latentserve_amd.kernels.hip import paged_sparse as ps
        for layer, pool in enumerate(self.k_pool):
            ps.rebuild_bounds(pool, self.kmin[layer], self.kmax[layer])

    def page_bounds(self, layer_idx: int):
        if self.kmin is None:
            return None
        return self.kmin[layer_idx], self.kmax[layer_idx]

    def _bound_pages(self, seq: int, first: int) -> None:
        """Bounds of a sequence's pages from `first` on, over the rows that it holds."""
        if self.kmin is None:
            return
        t = self.tables[seq]
        full = t.length // self.block_size
        if full > first:
            blks = torch.tensor(t.blocks[first:full]).to(self.device)
            for layer, pool in enumerate(self.k_pool):
                live = pool[blks]
                self.kmin[layer][blks] = live.amin(dim=1)
                self.kmax[layer][blks] = live.amax(dim=1)
        if t.length % self.block_size and full >= first:
            self._bound_partial_page(seq, t.length)

    def _bound_partial_page(self, seq: int, length: int) -> None:
        """Bounds of the page a rewind lands in, over its remaining rows."""
        t = self.tables[seq]
        page, rows = divmod(length, self.block_size)
        blk = t.blocks[page]
        for layer, pool in enumerate(self.k_pool):
            live = pool[blk, :rows]
            self.kmin[layer][blk] = live.amin(dim=0)
            self.kmax[layer][blk] = live.amax(dim=0)
