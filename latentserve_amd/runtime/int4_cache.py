"""4-bit paged KV cache for the HIP decode path.

The bookkeeping of the fp16 cache (tables, lengths, write slots at fixed
addresses, shared and copied pages) over the pools of kernels/hip/int4_cache.py:
160 bytes a token and KV head, against 512 in fp16.  An entry depends on its
token alone, so there is no residual as the INT8 cache has: a decode step's
write is one launch at published slots (capturable), a sequence can be rewound
to any token, and a partly filled page can be shared or copied.

Quantization runs on the HIP kernels only; there is no CPU path.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from latentserve_amd.runtime.kv_cache import KVCacheSpec, _PagedBase


class Int4PagedKVCache(_PagedBase):
    """4-bit paged KV storage."""

    def __init__(self, spec: KVCacheSpec, block_size: int = 16, num_blocks: Optional[int] = None):
        from latentserve_amd.kernels.hip import int4_cache as i4

        if spec.head_dim != i4.HEAD_DIM or spec.dtype != torch.float16:
            raise ValueError(f"the 4-bit cache holds float16 values of {i4.HEAD_DIM} channels, "
                             f"not {spec.dtype} of {spec.head_dim}")
        super().__init__(spec, block_size, num_blocks)
        self.pools = [i4.empty_pools(self.num_blocks, spec.num_kv_heads, self.device)
                      for _ in range(spec.num_layers)]

    def _page_tensors(self) -> List[torch.Tensor]:
        return [t for pools in self.pools for t in pools]

    def advance(self, n: int, batch_size: Optional[int] = None,
                slots: Optional[Sequence[int]] = None) -> None:
        """Reserve n more tokens for each active sequence and publish the
        step's kernel inputs.  OutOfBlocks leaves everything as it was."""
        self._room_for_step(n, batch_size, slots)
        self._publish(n, self._grow(n))

    def rewind(self, length: int, slots: Optional[Sequence[int]] = None) -> None:
        """Shorten sequences to `length` tokens, keeping their pages."""
        self._shorten(length, self._active if slots is None else list(slots))
        self._publish(0, [self.tables[s].length for s in self._active])

    def write(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, start_pos: int = 0) -> None:
        """Quantize k, v [B, H_kv, n, D] fp16 into the tokens the last advance(n)
        reserved."""
        from latentserve_amd.kernels.hip import int4_cache as i4

        b, _, n, _ = k.shape
        i4.write(k, v, self._slots_for_write(b, n).reshape(-1), self.pools[layer_idx])

    def read(self, layer_idx: int, batch_size: int, length: Optional[int] = None):
        """[B, H_kv, L, D] K and V of the active sequences, as the values their
        entries stand for (zeros past a sequence's end)."""
        from latentserve_amd.kernels.hip import int4_cache as i4

        length = self.max_len if length is None else length
        return i4.read(self.pools[layer_idx], self.block_tables_tensor(batch_size),
                       self.seq_lens_tensor(batch_size), length)
