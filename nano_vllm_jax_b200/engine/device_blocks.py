"""Block tables that grow on the device: a free list of block ids on the GPU and the rows' tables filled from it.

The reference's scheduler assigns blocks on the host and ships tables and slots with every step
(nanovllm_jax/engine/scheduler.py:734-1098).  `DeviceBlockPool` keeps the list where the tables are: `extend()` gives every row
the blocks that its new tokens need and returns the step's packed arrays, in one launch and without a copy from the host
(`kernels/paged_kv.py::build_packed_layout`).  The host only has to know the lengths' sum, for the token bucket.

The pool only hands out; ids come back by `reset()` with the ids that are free then, as the host's own bookkeeping knows them.
List and head stay where they are, so that a captured step goes on from where the one before it has left the list.
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
        """Start over with these ids (a sequence or an int32 tensor); the list's head goes back to its start.

        They take the place of the ids before, with -1 behind them where they are fewer; more than there ever were go into a new list, and
        steps that were captured with the old one have to be captured again."""
        ids = torch.as_tensor(free_blocks, dtype=torch.int32)
        if ids.ndim != 1:
            raise ValueError("free_blocks must be one-dimensional")
        n = ids.numel()
        if self.free_blocks is None or n > self.free_blocks.numel():
            self.free_blocks = torch.empty(n, dtype=torch.int32, device=self.device)
            self.free_head = torch.empty(1, dtype=torch.int32, device=self.device)
        self.free_blocks[:n].copy_(ids)
        self.free_blocks[n:].fill_(-1)
        self.free_head.zero_()

    def extend(self, block_tables, cached_lens, new_lens, token_bucket: int) -> _k.PackedLayout:
        """Room for `new_lens` more tokens behind `cached_lens` in every row of `block_tables` (in place), and the packed step's arrays.

        The list's head moves on with the call, in place: a captured call takes other ids at every replay.  A list that ends too early is flagged on
        the device (`check_device_status`)."""
        layout = _k.build_packed_layout(cached_lens, new_lens, block_tables, self.free_blocks, self.free_head, self.block_size, token_bucket)
        self.free_head.copy_(layout.free_head)
        return layout
