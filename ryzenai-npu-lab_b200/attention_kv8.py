"""Attention over the 8-bit paged cache (include/b2_kv8.h): torch-facing
wrappers and the PagedDecodeAttentionKV8 runner.

The cache holds e4m3 codes with a power-of-two scale for each block of 64
tokens and KV head (paged_cache.PagedKVCache8).  As in attention.py, host
checks raise ValueError, library refusals raise B2Error, work is queued on
the current CUDA stream of the tensors' device, and faults that only the
device sees (a bad block id, a length beyond the block table) are collected
in the caller's `dev_err` word.

    decode_step_kv8   append + attention of 1 to 4 new tokens per sequence
    append_kv8        q/k norm + RoPE + quantised append of a chunk
    prefill_kv8       append + attention of a prompt chunk, padded or packed
"""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from .attention import D, EPS, HKV, HQ, MAX_STEP_TOKENS, QKV_WIDTH, SCALE, _need, _need_rope
from .paged_cache import BLOCK, PagedKVCache8
from .rope import rope_table

NORM_ROPE_STORE = _lib.B2_NORM_QK | _lib.B2_ROPE_QK | _lib.B2_STORE_KV


def _on(device: torch.device):
    """Launches go to the current device: make it the tensors' own."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _raw_stream(device: torch.device, stream: torch.cuda.Stream | None) -> int:
    return (stream if stream is not None else torch.cuda.current_stream(device)).cuda_stream


def _addr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _is(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, shape: tuple) -> None:
    """_need with the checks that pass made cheap."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != shape or \
            not t.is_contiguous():
        _need(t, name, dtype, device, shape)


def _need_cache(k_pool, v_pool, k_scale, v_scale, device: torch.device) -> int:
    blocks = k_pool.shape[0] if isinstance(k_pool, torch.Tensor) and k_pool.dim() == 4 else 0
    _is(k_pool, "k_pool", torch.float8_e4m3fn, device, (blocks, HKV, BLOCK, D))
    _is(v_pool, "v_pool", torch.float8_e4m3fn, device, (blocks, HKV, D, BLOCK))
    _is(k_scale, "k_scale", torch.float32, device, (blocks, HKV))
    _is(v_scale, "v_scale", torch.float32, device, (blocks, HKV))
    return blocks


def _need_tables(block_tables, past_lens, chunk_lens, device: torch.device) -> tuple[int, int]:
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be [batch, max_blocks_per_seq]")
    b, width = block_tables.shape
    _is(block_tables, "block_tables", torch.int32, device, (b, width))
    _is(past_lens, "past_lens", torch.int32, device, (b,))
    if chunk_lens is not None:
        _is(chunk_lens, "chunk_lens", torch.int32, device, (b,))
    return b, width


def _need_qk(mode: int, gamma_q, gamma_k, cos, sin, device: torch.device) -> int:
    if mode & _lib.B2_NORM_QK:
        _is(gamma_q, "gamma_q", torch.bfloat16, device, (D,))
        _is(gamma_k, "gamma_k", torch.bfloat16, device, (D,))
    return _need_rope(cos, sin, device) if mode & _lib.B2_ROPE_QK else 0


def _need_workspace(workspace, device: torch.device) -> int:
    if not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 or workspace.device != device or \
            not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {device} (workspace_kv8)")
    return workspace.numel()


def workspace_kv8(device: torch.device | str) -> torch.Tensor:
    """The workspace of the 8-bit attention calls on `device`, zeroed.  Calls
    that share one must not overlap on the GPU; a captured graph and eager
    calls may share one as long as they run in turn."""
    return torch.zeros(_lib.load().b2_kv8_workspace_bytes(), dtype=torch.uint8, device=device)


def append_kv8(qkv: torch.Tensor, *, k_pool: torch.Tensor | None = None, v_pool: torch.Tensor | None = None,
               k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, dev_err: torch.Tensor,
               slots: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               past_lens: torch.Tensor | None = None, block_tables: torch.Tensor | None = None,
               chunk_lens: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
               gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, mode: int = NORM_ROPE_STORE,
               eps: float = EPS, stream: torch.cuda.Stream | None = None) -> None:
    """q/k RMSNorm + RoPE and the quantised append of k, v (b2_kv8_append).
    qkv: bf16 [rows, >= 2048] with `slots` int32 [rows] (and `positions` for
    RoPE) as the table builder writes them, a negative slot skipping its row;
    or [batch, tokens, >= 2048] with past_lens and block_tables.  q_out: bf16
    [rows, 16, 64] normalised and rotated query."""
    if not isinstance(qkv, torch.Tensor) or qkv.dim() not in (2, 3) or qkv.shape[-1] < QKV_WIDTH:
        raise ValueError(f"qkv must be [rows or batch x tokens, >= {QKV_WIDTH}]")
    dev = qkv.device
    _need(qkv, "qkv", torch.bfloat16, dev)
    width = qkv.shape[-1]
    rows = qkv.numel() // width
    tokens = table_width = 0
    if slots is not None:
        _is(slots, "slots", torch.int32, dev, (rows,))
        if positions is not None:
            _is(positions, "positions", torch.int32, dev, (rows,))
    else:
        if qkv.dim() != 3:
            raise ValueError("without slots, qkv must be [batch, tokens, width]")
        b, table_width = _need_tables(block_tables, past_lens, chunk_lens, dev)
        tokens = qkv.shape[1]
        if b != qkv.shape[0]:
            raise ValueError(f"block_tables must have {qkv.shape[0]} rows, got {b}")
    blocks = _need_cache(k_pool, v_pool, k_scale, v_scale, dev) if mode & _lib.B2_STORE_KV or slots is not None else 0
    if q_out is not None:
        _is(q_out, "q_out", torch.bfloat16, dev, (rows, HQ, D))
    rope_rows = _need_qk(mode, gamma_q, gamma_k, cos, sin, dev)
    _need(dev_err, "dev_err", torch.int32, dev)
    with _on(dev):
        rc = _lib.load().b2_kv8_append(
            qkv.data_ptr(), width, rows, _addr(slots), _addr(positions), _addr(past_lens), _addr(chunk_lens), tokens,
            _addr(block_tables), table_width, _addr(gamma_q), _addr(gamma_k), eps, _addr(cos), _addr(sin), rope_rows,
            _addr(k_pool), _addr(v_pool), _addr(k_scale), _addr(v_scale), blocks, _addr(q_out), mode,
            dev_err.data_ptr(), _raw_stream(dev, stream))
    _lib.check(rc, "b2_kv8_append")


def decode_step_kv8(qkv: torch.Tensor, past_lens: torch.Tensor, *, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor, out: torch.Tensor,
                    workspace: torch.Tensor, dev_err: torch.Tensor, chunk_lens: torch.Tensor | None = None,
                    gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None,
                    cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, mode: int = NORM_ROPE_STORE,
                    eps: float = EPS, scale: float = SCALE, stream: torch.cuda.Stream | None = None) -> None:
    """One decode step over the 8-bit cache (b2_kv8_decode_step): qkv bf16
    [B, T, >= 2048] raw projections of T = 1 to 4 new tokens per sequence at
    positions past_lens[b] + t, chunk_lens[b] (0 to T; None: T) of them there.
    Appends their k/v and writes the contexts into out [B, T, 16, 64]; rows
    past a sequence's chunk stay as they were.  `mode` as decode_step's."""
    if not isinstance(qkv, torch.Tensor) or qkv.dim() != 3 or qkv.shape[2] < QKV_WIDTH:
        raise ValueError(f"qkv must be [batch, tokens, >= {QKV_WIDTH}]")
    dev = qkv.device
    b, t, width = qkv.shape
    if not 1 <= t <= MAX_STEP_TOKENS:
        raise ValueError(f"tokens must be in [1, {MAX_STEP_TOKENS}], got {t}")
    _is(qkv, "qkv", torch.bfloat16, dev, (b, t, width))
    tb, table_width = _need_tables(block_tables, past_lens, chunk_lens, dev)
    if tb != b:
        raise ValueError(f"block_tables must have {b} rows, got {tb}")
    blocks = _need_cache(k_pool, v_pool, k_scale, v_scale, dev)
    _is(out, "out", torch.bfloat16, dev, (b, t, HQ, D))
    _need(dev_err, "dev_err", torch.int32, dev)
    rope_rows = _need_qk(mode, gamma_q, gamma_k, cos, sin, dev)
    nbytes = _need_workspace(workspace, dev)
    with _on(dev):
        rc = _lib.load().b2_kv8_decode_step(
            qkv.data_ptr(), width, t, _addr(chunk_lens), _addr(gamma_q), _addr(gamma_k), eps, _addr(cos), _addr(sin),
            rope_rows, past_lens.data_ptr(), block_tables.data_ptr(), table_width, k_pool.data_ptr(),
            v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, b, scale, mode, out.data_ptr(),
            workspace.data_ptr(), nbytes, dev_err.data_ptr(), _raw_stream(dev, stream))
    _lib.check(rc, "b2_kv8_decode_step")


def prefill_kv8(qkv: torch.Tensor, past_lens: torch.Tensor, *, k_pool: torch.Tensor, v_pool: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor, workspace: torch.Tensor,
                dev_err: torch.Tensor, chunk_lens: torch.Tensor | None = None, row_start: torch.Tensor | None = None,
                max_tokens: int | None = None, slots: torch.Tensor | None = None,
                positions: torch.Tensor | None = None, gamma_q: torch.Tensor | None = None,
                gamma_k: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                sin: torch.Tensor | None = None, mode: int = NORM_ROPE_STORE, eps: float = EPS, scale: float = SCALE,
                out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """A prompt chunk over the 8-bit cache: append (b2_kv8_append), then
    attention of every new token over the cache up to itself
    (b2_kv8_prefill_attn).

    Padded: qkv bf16 [B, T, >= 2048], token t of sequence b at position
    past_lens[b] + t, chunk_lens[b] <= T of them there.
    Packed: qkv bf16 [rows, >= 2048], sequence b's chunk_lens[b] <= max_tokens
    tokens from row row_start[b] on, with the slots (and positions) that
    block_tables.extend_tables or slot_map wrote for the rows.

    Returns the contexts [rows, 16, 64] ([B, T, 16, 64] for padded qkv) in
    `out` when given; rows of no token stay as they were (zero without `out`)."""
    if not isinstance(qkv, torch.Tensor) or qkv.dim() not in (2, 3) or qkv.shape[-1] < QKV_WIDTH:
        raise ValueError(f"qkv must be [rows, >= {QKV_WIDTH}] or [batch, tokens, >= {QKV_WIDTH}]")
    dev = qkv.device
    width = qkv.shape[-1]
    rows = qkv.numel() // width
    b, table_width = _need_tables(block_tables, past_lens, chunk_lens, dev)
    if qkv.dim() == 3:
        tokens = qkv.shape[1]
        if qkv.shape[0] != b or row_start is not None:
            raise ValueError(f"padded qkv must be [{b}, tokens, width], without row_start")
        shape = (b, tokens, HQ, D)
    else:
        if row_start is None or max_tokens is None or slots is None:
            raise ValueError("packed qkv needs row_start, max_tokens and slots")
        _is(row_start, "row_start", torch.int32, dev, (b,))
        tokens = int(max_tokens)
        shape = (rows, HQ, D)
    if out is None:
        out = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
    _is(out, "out", torch.bfloat16, dev, shape)
    blocks = _need_cache(k_pool, v_pool, k_scale, v_scale, dev)
    nbytes = _need_workspace(workspace, dev)
    turned = mode & (_lib.B2_NORM_QK | _lib.B2_ROPE_QK)
    q = torch.empty(rows, HQ, D, dtype=torch.bfloat16, device=dev) if turned else None
    if mode:
        append_kv8(qkv, k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, dev_err=dev_err, slots=slots,
                   positions=positions, past_lens=past_lens, block_tables=block_tables, chunk_lens=chunk_lens,
                   q_out=q, gamma_q=gamma_q, gamma_k=gamma_k, cos=cos, sin=sin, mode=mode, eps=eps, stream=stream)
    else:
        _need(qkv, "qkv", torch.bfloat16, dev)
        _need(dev_err, "dev_err", torch.int32, dev)
    with _on(dev):
        rc = _lib.load().b2_kv8_prefill_attn(
            qkv.data_ptr() if q is None else q.data_ptr(), width if q is None else HQ * D, rows, _addr(row_start),
            past_lens.data_ptr(), _addr(chunk_lens), tokens, block_tables.data_ptr(), table_width, k_pool.data_ptr(),
            v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, b, scale, out.data_ptr(),
            workspace.data_ptr(), nbytes, dev_err.data_ptr(), _raw_stream(dev, stream))
    _lib.check(rc, "b2_kv8_prefill_attn")
    return out


class PagedDecodeAttentionKV8:
    """PagedDecodeAttention over a PagedKVCache8: step() runs one decode step of
    1 to 4 new tokens per sequence, prefill() a prompt chunk.  The workspace is
    allocated here once; step() allocates nothing and can be captured in a CUDA
    graph.  Calls of one runner must not overlap on the GPU."""

    def __init__(self, cache: PagedKVCache8, gamma_q: torch.Tensor, gamma_k: torch.Tensor, max_batch: int,
                 rope_positions: int, *, max_tokens: int = 1, eps: float = EPS, scale: float = SCALE,
                 workspace: torch.Tensor | None = None):
        if not isinstance(cache, PagedKVCache8):
            raise ValueError("cache must be a PagedKVCache8")
        self.cache, self.device, self.eps, self.scale = cache, cache.device, eps, scale
        dev = cache.k.device
        self.gamma_q = gamma_q.to(dev, torch.bfloat16).contiguous()
        self.gamma_k = gamma_k.to(dev, torch.bfloat16).contiguous()
        self.cos, self.sin = rope_table(rope_positions, device=dev)
        self.max_batch = max_batch
        self.out = torch.zeros(max_batch * max_tokens, HQ, D, dtype=torch.bfloat16, device=dev)
        self.workspace = workspace if workspace is not None else workspace_kv8(dev)
        self.dev_err = torch.zeros(1, dtype=torch.int32, device=dev)

    def _common(self, layer: int) -> dict:
        return {**self.cache.kv8(layer), "workspace": self.workspace, "dev_err": self.dev_err, "gamma_q": self.gamma_q,
                "gamma_k": self.gamma_k, "cos": self.cos, "sin": self.sin, "eps": self.eps, "scale": self.scale}

    def step(self, layer: int, qkv: torch.Tensor, past_lens: torch.Tensor, block_tables: torch.Tensor, *,
             chunk_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
             stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """qkv bf16 [B, W] (one token per sequence) or [B, T, W] raw projections;
        returns the contexts [B, 16, 64] or [B, T, 16, 64]."""
        rows = qkv if qkv.dim() == 3 else qkv.unsqueeze(1)
        b, t = rows.shape[:2]
        if out is None:
            if b * t > self.out.shape[0]:
                raise ValueError(f"{b} x {t} tokens > max_batch x max_tokens {self.out.shape[0]}")
            out = self.out[:b * t].view(b, t, HQ, D) if qkv.dim() == 3 else self.out[:b]
        decode_step_kv8(rows, past_lens, block_tables=block_tables, chunk_lens=chunk_lens, out=out.view(b, t, HQ, D),
                        stream=stream, **self._common(layer))
        return out

    def prefill(self, layer: int, qkv: torch.Tensor, past_lens: torch.Tensor, block_tables: torch.Tensor,
                **chunk) -> torch.Tensor:
        """prefill_kv8 of one layer with the runner's norm weights and RoPE tables."""
        return prefill_kv8(qkv, past_lens, block_tables=block_tables, **chunk, **self._common(layer))

    def check(self) -> None:
        """Synchronise on the device error word; raise if any kernel flagged one."""
        word = int(self.dev_err.item())
        if word:
            self.dev_err.zero_()
            self.workspace.zero_()   # an aborted step may leave counts behind
            raise RuntimeError("8-bit decode attention device error: " + "; ".join(_lib.decode_dev_err(word)))
