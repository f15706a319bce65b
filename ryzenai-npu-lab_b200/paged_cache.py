"""Paged BF16 KV cache: block pools, a block allocator and block tables.

Replaces the reference's per-core cache buffers, which are copied whole on
every append (experiments/kernels/lfm25_attention_append_cache.cc:5-39) or
streamed at a fixed capacity tier (experiments/lfm25_x8.py:116-123,263-270;
experiments/lfm25_x8_model.py:22,139).

Layout per attention layer (the library's pool layout):
    k_pool, v_pool : bf16 [num_blocks, 8 kv heads, 64 tokens, 64 dims]
One (block, head) tile is 8 KiB contiguous, which is the unit the decode
kernel streams with one TMA box.  Token t of a sequence lives in pool block
block_table[t // 64], row t % 64.  All layers share the block tables (a
sequence owns the same block ids in every layer's pool).
"""
from __future__ import annotations

import torch

HKV, D, BLOCK = 8, 64, 64
BLOCK_BYTES = 2 * HKV * BLOCK * D * 2   # K + V tile bytes of one block, all heads: 128 KiB


def blocks_for(tokens: int) -> int:
    return (tokens + BLOCK - 1) // BLOCK


class BlockAllocator:
    """Free list of pool block ids (host side).  The order of the free list is
    shuffled with a seeded generator when `shuffle_seed` is given, so that a
    sequence's blocks are scattered over the pool like in a long-running server."""

    def __init__(self, num_blocks: int, shuffle_seed: int | None = None):
        if num_blocks <= 0:
            raise ValueError("num_blocks must be positive")
        self.num_blocks = num_blocks
        if shuffle_seed is None:
            order = list(range(num_blocks))
        else:
            g = torch.Generator().manual_seed(shuffle_seed)
            order = torch.randperm(num_blocks, generator=g).tolist()
        self._free = order[::-1]   # pop() hands out order[0], order[1], ...
        self._used: set[int] = set()

    @property
    def free(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> list[int]:
        if n < 0:
            raise ValueError("n must be >= 0")
        if n > len(self._free):
            raise MemoryError(f"KV pool exhausted: need {n} blocks, {len(self._free)} free")
        out = [self._free.pop() for _ in range(n)]
        self._used.update(out)
        return out

    def release(self, blocks) -> None:
        """Return blocks to the free list.  A block outside the pool, not
        handed out, or listed twice is refused (nothing is released): two
        sequences sharing a block would overwrite each other's keys."""
        blocks = list(blocks)
        for b in blocks:
            if not 0 <= b < self.num_blocks:
                raise ValueError(f"block {b} outside the pool")
            if b not in self._used:
                raise ValueError(f"block {b} is not allocated")
        if len(set(blocks)) != len(blocks):
            raise ValueError("a block is listed twice")
        self._used.difference_update(blocks)
        self._free.extend(blocks)


class PagedKVCache:
    """K/V pools for `num_layers` attention layers plus per-sequence block tables.

    capacity_tokens is the most tokens any sequence may hold; it fixes the
    block-table width (max_blocks_per_seq).  Sequences are registered with
    `add_sequence`, which allocates the blocks its capacity needs up front, so
    a decode step never allocates.
    """

    def __init__(self, num_blocks: int, capacity_tokens: int, num_layers: int = 1,
                 device: torch.device | str = "cuda", shuffle_seed: int | None = None,
                 fill: float | None = None):
        if capacity_tokens <= 0:
            raise ValueError("capacity_tokens must be positive")
        self.num_blocks = num_blocks
        self.num_layers = num_layers
        self.device = torch.device(device)
        self.max_blocks = blocks_for(capacity_tokens)
        self._allocate((num_layers, num_blocks, HKV, BLOCK, D), fill)
        self.allocator = BlockAllocator(num_blocks, shuffle_seed)
        self._tables: list[list[int]] = []
        self.lengths: list[int] = []

    def _allocate(self, shape, fill: float | None) -> None:
        if fill is None:
            self.k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
            self.v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        else:
            self.k = torch.full(shape, fill, dtype=torch.bfloat16, device=self.device)
            self.v = torch.full(shape, fill, dtype=torch.bfloat16, device=self.device)

    @property
    def batch(self) -> int:
        return len(self._tables)

    def add_sequence(self, length: int = 0, capacity: int | None = None) -> int:
        cap = self.max_blocks * BLOCK if capacity is None else capacity
        if not 0 <= length <= cap <= self.max_blocks * BLOCK:
            raise ValueError(f"length {length} / capacity {cap} outside [0, {self.max_blocks * BLOCK}]")
        self._tables.append(self.allocator.alloc(blocks_for(cap)))
        self.lengths.append(length)
        return len(self._tables) - 1

    def release_sequence(self, seq: int) -> None:
        """Return a finished sequence's blocks to the pool.  Its row stays (block
        tables keep their batch index) with no blocks and length 0: it must
        not be stepped again, since a row of -1 entries is a device error."""
        self.allocator.release(self._tables[seq])
        self._tables[seq] = []
        self.lengths[seq] = 0

    def block_tables(self) -> torch.Tensor:
        """int32 [batch, max_blocks_per_seq]; unused entries are -1."""
        t = torch.full((self.batch, self.max_blocks), -1, dtype=torch.int32)
        for i, row in enumerate(self._tables):
            t[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
        return t.to(self.device)

    def table(self, seq: int) -> list[int]:
        return list(self._tables[seq])

    def pool(self, layer: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
        return self.k[layer], self.v[layer]

    def write_dense(self, layer: int, seq: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Copy a dense [8, T, 64] history into the sequence's blocks (set-up
        of synthetic caches and of the reference-layout shims; not the decode path)."""
        t = k.shape[1]
        if blocks_for(t) > len(self._tables[seq]):
            raise ValueError("history longer than the sequence's capacity")
        kp, vp = self.pool(layer)
        nb = blocks_for(t)
        if nb == 0:
            return
        ids = torch.tensor(self._tables[seq][:nb], device=self.device)
        pad = nb * BLOCK - t
        kd = torch.nn.functional.pad(k.to(self.device), (0, 0, 0, pad)).reshape(HKV, nb, BLOCK, D)
        vd = torch.nn.functional.pad(v.to(self.device), (0, 0, 0, pad)).reshape(HKV, nb, BLOCK, D)
        kp[ids] = kd.transpose(0, 1).to(torch.bfloat16)
        vp[ids] = vd.transpose(0, 1).to(torch.bfloat16)

    def read_dense(self, layer: int, seq: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """[8, length, 64] K and V of one sequence (the x8 runner's kv(),
        experiments/lfm25_x8_model.py:85-92)."""
        kp, vp = self.pool(layer)
        nb = blocks_for(length)
        ids = torch.tensor(self._tables[seq][:nb], device=self.device, dtype=torch.long)
        k = kp[ids].transpose(0, 1).reshape(HKV, nb * BLOCK, D)[:, :length]
        v = vp[ids].transpose(0, 1).reshape(HKV, nb * BLOCK, D)[:, :length]
        return k, v


KV8_MAX = 448.0              # the largest e4m3 code
KV8_MIN_SCALE = 2.0 ** -100


def kv8_scale(amax: torch.Tensor) -> torch.Tensor:
    """The scale of a (block, head) whose largest magnitude is `amax` (finite,
    >= 0): the smallest power of two s >= 2^-100 with amax <= 448 * s."""
    m, e = torch.frexp(amax.float() / KV8_MAX)
    s = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e))
    return torch.where(amax > 0, s, torch.zeros_like(s)).clamp(min=KV8_MIN_SCALE)


class PagedKVCache8(PagedKVCache):
    """PagedKVCache in 8 bits: e4m3 codes with a power-of-two fp32 scale for
    each block and KV head, half the bytes of the bf16 cache.

        k        float8_e4m3fn [layers, num_blocks, 8, 64 tokens, 64 dims]
        v        float8_e4m3fn [layers, num_blocks, 8, 64 dims, 64 tokens]
        k_scale, v_scale       float32 [layers, num_blocks, 8]

    A block's scale follows its largest value and never falls while the block
    holds tokens: after a shorter length (drafted tokens that were rejected) the
    next append keeps the scale that they raised.

    attention_kv8 appends to it and attends over it; the bf16 kernels refuse
    it.  Block allocation and tables are PagedKVCache's."""

    def _allocate(self, shape, fill: float | None) -> None:
        layers, blocks = shape[:2]
        tiles = (layers, blocks, HKV, BLOCK * D)

        def codes():
            if fill is None:
                return torch.empty(tiles, dtype=torch.float8_e4m3fn, device=self.device)
            return torch.full(tiles, fill, dtype=torch.float32).to(torch.float8_e4m3fn).to(self.device)
        self.k = codes().view(layers, blocks, HKV, BLOCK, D)
        self.v = codes().view(layers, blocks, HKV, D, BLOCK)
        value = 1.0 if fill is None else fill
        self.k_scale = torch.full((layers, blocks, HKV), value, dtype=torch.float32, device=self.device)
        self.v_scale = torch.full((layers, blocks, HKV), value, dtype=torch.float32, device=self.device)

    def kv8(self, layer: int = 0) -> dict[str, torch.Tensor]:
        """The layer's pools and scales under the names attention_kv8 takes."""
        return {"k_pool": self.k[layer], "v_pool": self.v[layer], "k_scale": self.k_scale[layer],
                "v_scale": self.v_scale[layer]}

    def write_dense(self, layer: int, seq: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantise a dense [8, T, 64] history into the sequence's blocks (set-up,
        not the decode path): what one append of the T tokens to the empty
        sequence stores."""
        t = k.shape[1]
        nb = blocks_for(t)
        if nb > len(self._tables[seq]):
            raise ValueError("history longer than the sequence's capacity")
        if nb == 0:
            return
        ids = torch.tensor(self._tables[seq][:nb], device=self.device)
        pad = nb * BLOCK - t
        for x, pool, scale, dim_major in ((k, self.k, self.k_scale, False), (v, self.v, self.v_scale, True)):
            x = torch.nn.functional.pad(x.to(self.device, torch.bfloat16).float(), (0, 0, 0, pad))
            x = x.reshape(HKV, nb, BLOCK, D).transpose(0, 1)
            big = torch.finfo(torch.bfloat16).max
            x = x.clamp(-big, big)
            s = kv8_scale(x.abs().nan_to_num(0.0).amax((2, 3)))
            c = (x / s[..., None, None]).to(torch.float8_e4m3fn)
            c = c.transpose(2, 3) if dim_major else c
            pool[layer].view(torch.uint8)[ids] = c.contiguous().view(torch.uint8)
            scale[layer][ids] = s

    def read_dense(self, layer: int, seq: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """[8, length, 64] bf16 K and V of one sequence, the values its codes
        stand for (bf16 holds a code times its scale exactly)."""
        return self.read_blocks(layer, self._tables[seq], length)

    def read_blocks(self, layer: int, blocks, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """read_dense of a sequence whose blocks are not this cache's own (a
        device block table's row)."""
        nb = blocks_for(length)
        ids = torch.as_tensor(blocks, device=self.device).long()[:nb]
        out = []
        for pool, scale, dim_major in ((self.k, self.k_scale, False), (self.v, self.v_scale, True)):
            x = pool[layer].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * scale[layer][ids][..., None, None]
            x = x.transpose(2, 3) if dim_major else x
            out.append(x.transpose(0, 1).reshape(HKV, nb * BLOCK, D)[:, :length].to(torch.bfloat16))
        return out[0], out[1]
