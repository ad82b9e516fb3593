"""Block tables that grow on the device: a free list of block ids on the GPU and the rows' tables filled from it.

The reference's scheduler assigns blocks on the host and ships tables and slots with every step
(nanovllm_jax/engine/scheduler.py:734-1098).  `DeviceBlockPool` keeps the list where the tables are: `extend()` gives every row
the blocks that its new tokens need and returns the step's packed arrays, in one launch and without a copy from the host
(`kernels/paged_kv.py::build_packed_layout`).  The host only has to know the lengths' sum, for the token bucket.

The pool only hands out; ids come back by `reset()` with the ids that are free then, as the host's own bookkeeping knows them.
"""

from __future__ import annotations

from typing import Optional

import torch

from ..kernels import paged_kv as _k


class DeviceBlockPool:
    """Free block ids on the device, handed out in order."""

    def __init__(self, free_blocks, block_size: int, device="cuda"):
        self.device = torch.device(device)
        self.block_size = int(block_size)
        if self.block_size <= 0:
            raise ValueError("block_size must be positive")
        self.free_blocks: Optional[torch.Tensor] = None
        self.reset(free_blocks)

    def reset(self, free_blocks) -> None:
        """Start over with these ids (a sequence or an int32 tensor); the list's head goes back to its start."""
        ids = torch.as_tensor(free_blocks, dtype=torch.int32)
        if ids.ndim != 1:
            raise ValueError("free_blocks must be one-dimensional")
        self.free_blocks = ids.to(self.device).contiguous()
        self.free_head = torch.zeros(1, dtype=torch.int32, device=self.device)

    def extend(self, block_tables, cached_lens, new_lens, token_bucket: int) -> _k.PackedLayout:
        """Room for `new_lens` more tokens behind `cached_lens` in every row of `block_tables` (in place), and the packed step's arrays.

        The list's head moves on with the call: a captured call takes the same ids at every replay, unless the caller copies
        `layout.free_head` into the tensor that was the pool's head before."""
        layout = _k.build_packed_layout(cached_lens, new_lens, block_tables, self.free_blocks, self.free_head, self.block_size, token_bucket)
        self.free_head = layout.free_head
        return layout
