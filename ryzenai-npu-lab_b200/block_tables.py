"""Block tables and slot maps built on the GPU (include/b2_tables.h).

PagedKVCache hands out blocks on the host and reserves a sequence's whole
capacity up front.  Here the tables live on the device and grow with the
requests: the blocks of new tokens are taken from a free list and the place of
every new token is written by kernels, so a scheduler needs no host round trip
and a decode loop can allocate inside a captured CUDA graph.

    extend_tables      blocks, grants, slots and positions for new tokens
    slot_map           slots and positions alone, from tables that are there
    release_tables     finished requests' blocks back to the free list
    DeviceBlockTables  the allocator that owns such tables
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .attention_kv8 import _addr, _is, _on, _raw_stream
from .paged_cache import blocks_for


def extend_tables(block_tables: torch.Tensor, held: torch.Tensor, free_list: torch.Tensor, free_count: torch.Tensor,
                  past_lens: torch.Tensor, new_lens: torch.Tensor, *, granted: torch.Tensor, row_start: torch.Tensor,
                  slots: torch.Tensor, positions: torch.Tensor, dev_err: torch.Tensor, tokens_per_seq: int = 0,
                  held_out: torch.Tensor | None = None, free_count_out: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None) -> None:
    """Blocks for new_lens[b] tokens behind past_lens[b] and the place of every
    new token (b2_tables_extend); all int32.  block_tables [B, width] gets the
    new entries, held_out [B] and free_count_out [1] (None: in place) the new
    state, granted [B] new_lens or 0 for a refused request, row_start [B] the
    first row of each, slots / positions [rows] the slot (block * 64 + row; -1
    for no token) and position of each row.  tokens_per_seq: 0 for packed rows,
    T for rows b * T + t."""
    dev = block_tables.device
    if block_tables.dim() != 2 or not isinstance(slots, torch.Tensor):
        raise ValueError("block_tables must be [batch, max_blocks_per_seq], slots a tensor")
    b, width = block_tables.shape
    rows = slots.numel()
    held_out = held if held_out is None else held_out
    free_count_out = free_count if free_count_out is None else free_count_out
    i32 = torch.int32
    _is(block_tables, "block_tables", i32, dev, (b, width))
    _is(held, "held", i32, dev, (b,))
    _is(free_list, "free_list", i32, dev, (free_list.numel(),))
    _is(free_count, "free_count", i32, dev, (1,))
    _is(past_lens, "past_lens", i32, dev, (b,))
    _is(new_lens, "new_lens", i32, dev, (b,))
    _is(held_out, "held_out", i32, dev, (b,))
    _is(free_count_out, "free_count_out", i32, dev, (1,))
    _is(granted, "granted", i32, dev, (b,))
    _is(row_start, "row_start", i32, dev, (b,))
    _is(slots, "slots", i32, dev, (rows,))
    _is(positions, "positions", i32, dev, (rows,))
    _is(dev_err, "dev_err", i32, dev, (1,))
    with _on(dev):
        rc = _lib.load().b2_tables_extend(
            block_tables.data_ptr(), width, held.data_ptr(), free_list.data_ptr(), free_list.numel(),
            free_count.data_ptr(), past_lens.data_ptr(), new_lens.data_ptr(), b, held_out.data_ptr(),
            free_count_out.data_ptr(), granted.data_ptr(), row_start.data_ptr(), slots.data_ptr(),
            positions.data_ptr(), rows, tokens_per_seq, dev_err.data_ptr(), _raw_stream(dev, stream))
    _lib.check(rc, "b2_tables_extend")


def slot_map(block_tables: torch.Tensor, past_lens: torch.Tensor, new_lens: torch.Tensor, *, num_blocks: int,
             slots: torch.Tensor, positions: torch.Tensor, dev_err: torch.Tensor,
             row_start: torch.Tensor | None = None, tokens_per_seq: int = 0,
             stream: torch.cuda.Stream | None = None) -> None:
    """Slots and positions of new_lens[b] tokens behind past_lens[b] from tables
    whose blocks are there (b2_slot_map): rows from row_start[b] on (ascending,
    not overlapping), or rows b * tokens_per_seq + t."""
    dev = block_tables.device
    if block_tables.dim() != 2 or not isinstance(slots, torch.Tensor):
        raise ValueError("block_tables must be [batch, max_blocks_per_seq], slots a tensor")
    b, width = block_tables.shape
    rows = slots.numel()
    i32 = torch.int32
    _is(block_tables, "block_tables", i32, dev, (b, width))
    _is(past_lens, "past_lens", i32, dev, (b,))
    _is(new_lens, "new_lens", i32, dev, (b,))
    if row_start is not None:
        _is(row_start, "row_start", i32, dev, (b,))
    _is(slots, "slots", i32, dev, (rows,))
    _is(positions, "positions", i32, dev, (rows,))
    _is(dev_err, "dev_err", i32, dev, (1,))
    with _on(dev):
        rc = _lib.load().b2_slot_map(
            block_tables.data_ptr(), width, num_blocks, past_lens.data_ptr(), new_lens.data_ptr(), _addr(row_start),
            b, slots.data_ptr(), positions.data_ptr(), rows, tokens_per_seq, dev_err.data_ptr(),
            _raw_stream(dev, stream))
    _lib.check(rc, "b2_slot_map")


def release_tables(block_tables: torch.Tensor, held: torch.Tensor, free_list: torch.Tensor, free_count: torch.Tensor,
                   finished: torch.Tensor, *, dev_err: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
    """Blocks of the requests with finished[b] (bool [B]) back to the free list
    (b2_tables_release); their rows become -1 and held[b] 0."""
    dev = block_tables.device
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [batch, max_blocks_per_seq]")
    b, width = block_tables.shape
    _is(block_tables, "block_tables", torch.int32, dev, (b, width))
    _is(held, "held", torch.int32, dev, (b,))
    _is(free_list, "free_list", torch.int32, dev, (free_list.numel(),))
    _is(free_count, "free_count", torch.int32, dev, (1,))
    _is(finished, "finished", torch.bool, dev, (b,))
    _is(dev_err, "dev_err", torch.int32, dev, (1,))
    with _on(dev):
        rc = _lib.load().b2_tables_release(
            block_tables.data_ptr(), width, held.data_ptr(), free_list.data_ptr(), free_list.numel(),
            free_count.data_ptr(), finished.data_ptr(), b, dev_err.data_ptr(), _raw_stream(dev, stream))
    _lib.check(rc, "b2_tables_release")


@dataclass
class TokenPlan:
    """Where the new tokens of one step go (all int32 on the device)."""
    past: torch.Tensor        # [B] tokens cached before (the allocator's lengths, until advance())
    granted: torch.Tensor     # [B] new tokens, 0 for a request that got no blocks
    row_start: torch.Tensor   # [B] first row of each request
    slots: torch.Tensor       # [rows]
    positions: torch.Tensor   # [rows]


class DeviceBlockTables:
    """Allocator of a paged pool's blocks whose state lives on the GPU.

    tables [max_batch, width], held [max_batch], lens [max_batch] (tokens
    cached), a free list.  plan() takes the blocks of a step's new tokens,
    advance() counts them as cached once they are appended, release() returns
    finished requests' blocks.  All three only queue work on the current stream
    and can be captured in a CUDA graph."""

    def __init__(self, max_batch: int, num_blocks: int, capacity_tokens: int, device: torch.device | str = "cuda"):
        if max_batch <= 0 or num_blocks <= 0 or capacity_tokens <= 0:
            raise ValueError("max_batch, num_blocks and capacity_tokens must be positive")
        dev = torch.device(device)

        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=dev)
        self.num_blocks, self.max_batch = num_blocks, max_batch
        self.tables = ints(max_batch, blocks_for(capacity_tokens), value=-1)
        self.held, self.lens = ints(max_batch), ints(max_batch)
        # taken from the end: block 0 first
        self.free_list = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = ints(1, value=num_blocks)
        self.dev_err = ints(1)

    def plan(self, new_lens: torch.Tensor, *, rows: int | None = None, tokens_per_seq: int = 0,
             out: TokenPlan | None = None) -> TokenPlan:
        """Blocks and places for new_lens[b] new tokens: padded rows
        (tokens_per_seq = T) or packed into `rows` rows.  `out`: a plan of the
        same sizes to write into."""
        if out is None:
            n = self.max_batch * tokens_per_seq if tokens_per_seq > 0 else rows
            if n is None:
                raise ValueError("rows or tokens_per_seq > 0 is required")

            def ints(k):
                return torch.empty(k, dtype=torch.int32, device=self.tables.device)
            out = TokenPlan(self.lens, ints(self.max_batch), ints(self.max_batch), ints(n), ints(n))
        extend_tables(self.tables, self.held, self.free_list, self.free_count, self.lens, new_lens,
                      granted=out.granted, row_start=out.row_start, slots=out.slots, positions=out.positions,
                      tokens_per_seq=tokens_per_seq, dev_err=self.dev_err)
        return out

    def advance(self, plan: TokenPlan) -> None:
        """Count the plan's granted tokens as cached."""
        self.lens.add_(plan.granted)

    def release(self, finished: torch.Tensor) -> None:
        """Return the blocks of the requests with finished[b] (bool [max_batch])."""
        release_tables(self.tables, self.held, self.free_list, self.free_count, finished, dev_err=self.dev_err)
        self.lens.masked_fill_(finished, 0)

    def check(self) -> None:
        """Raise RuntimeError if a kernel flagged a bad length or block."""
        word = int(self.dev_err.item())
        if word:
            self.dev_err.zero_()
            raise RuntimeError("block table device error: " + "; ".join(_lib.decode_dev_err(word)))
