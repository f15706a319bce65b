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
from .attention_kv8 import _I32, _is, _launch, _native
from .paged_cache import blocks_for


def _table_shape(block_tables) -> torch.Size:
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be [batch, max_blocks_per_seq]")
    return block_tables.shape


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
    native, raw = _native(block_tables, stream)
    if native is not None:
        rc = native.extend(block_tables, held, free_list, free_count, past_lens, new_lens, held_out, free_count_out,
                           granted, row_start, slots, positions, tokens_per_seq, dev_err, raw)
        if rc == 0:
            return
        if rc is not None:
            _lib.check(rc, "b2_tables_extend")
    b, width = _table_shape(block_tables)
    rows, blocks = slots.numel(), free_list.numel()
    index, per_b = block_tables.get_device(), (b,)
    held_at = _is(held, "held", _I32, block_tables, index, per_b)
    count_at = _is(free_count, "free_count", _I32, block_tables, index, (1,))
    _launch("b2_tables_extend", index, stream,
            _is(block_tables, "block_tables", _I32, block_tables, index, (b, width)), width, held_at,
            _is(free_list, "free_list", _I32, block_tables, index, (blocks,)), blocks, count_at,
            _is(past_lens, "past_lens", _I32, block_tables, index, per_b),
            _is(new_lens, "new_lens", _I32, block_tables, index, per_b), b,
            held_at if held_out is None else _is(held_out, "held_out", _I32, block_tables, index, per_b),
            count_at if free_count_out is None else _is(free_count_out, "free_count_out", _I32, block_tables, index, (1,)),
            _is(granted, "granted", _I32, block_tables, index, per_b),
            _is(row_start, "row_start", _I32, block_tables, index, per_b),
            _is(slots, "slots", _I32, block_tables, index, (rows,)),
            _is(positions, "positions", _I32, block_tables, index, (rows,)), rows, tokens_per_seq,
            _is(dev_err, "dev_err", _I32, block_tables, index, (1,)))


def slot_map(block_tables: torch.Tensor, past_lens: torch.Tensor, new_lens: torch.Tensor, *, num_blocks: int,
             slots: torch.Tensor, positions: torch.Tensor, dev_err: torch.Tensor,
             row_start: torch.Tensor | None = None, tokens_per_seq: int = 0,
             stream: torch.cuda.Stream | None = None) -> None:
    """Slots and positions of new_lens[b] tokens behind past_lens[b] from tables
    whose blocks are there (b2_slot_map): rows from row_start[b] on (ascending,
    not overlapping), or rows b * tokens_per_seq + t.  A request whose lengths
    do not fit gets no slot at all (-1) and is flagged in dev_err."""
    b, width = _table_shape(block_tables)
    rows, index, per_b = slots.numel(), block_tables.get_device(), (b,)
    _launch("b2_slot_map", index, stream,
            _is(block_tables, "block_tables", _I32, block_tables, index, (b, width)), width, num_blocks,
            _is(past_lens, "past_lens", _I32, block_tables, index, per_b),
            _is(new_lens, "new_lens", _I32, block_tables, index, per_b),
            None if row_start is None else _is(row_start, "row_start", _I32, block_tables, index, per_b), b,
            _is(slots, "slots", _I32, block_tables, index, (rows,)),
            _is(positions, "positions", _I32, block_tables, index, (rows,)), rows, tokens_per_seq,
            _is(dev_err, "dev_err", _I32, block_tables, index, (1,)))


def release_tables(block_tables: torch.Tensor, held: torch.Tensor, free_list: torch.Tensor, free_count: torch.Tensor,
                   finished: torch.Tensor, *, dev_err: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
    """Blocks of the requests with finished[b] (bool [B]) back to the free list
    (b2_tables_release); their rows become -1 and held[b] 0."""
    b, width = _table_shape(block_tables)
    index, blocks = block_tables.get_device(), free_list.numel()
    _launch("b2_tables_release", index, stream,
            _is(block_tables, "block_tables", _I32, block_tables, index, (b, width)), width,
            _is(held, "held", _I32, block_tables, index, (b,)),
            _is(free_list, "free_list", _I32, block_tables, index, (blocks,)), blocks,
            _is(free_count, "free_count", _I32, block_tables, index, (1,)),
            _is(finished, "finished", torch.bool, block_tables, index, (b,)), b,
            _is(dev_err, "dev_err", _I32, block_tables, index, (1,)))


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
