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

import ctypes

import torch

from . import _lib
from .attention import D, EPS, HKV, HQ, MAX_STEP_TOKENS, QKV_WIDTH, SCALE, _need, _need_rope
from .build import binding_matches
from .paged_cache import BLOCK, PagedKVCache8
from .rope import rope_table

NORM_ROPE_STORE = _lib.B2_NORM_QK | _lib.B2_ROPE_QK | _lib.B2_STORE_KV


# The smallest calls are bound by the host.  The native binding (_b2torch, built
# against the installed torch) checks a call's tensors and makes the library call
# in one go, in half the time; where it is not built (or for another torch), or says None to
# an argument, the checks below do the same: each is one comparison of what the tensor says about itself
# (its device by index), and the slow path that words the refusal is taken only
# when one fails.
_b2torch = None
if binding_matches():
    try:
        from . import _b2torch
    except ImportError:
        pass
_bound = None       # the library whose functions the binding holds


def _native(t, stream: torch.cuda.Stream | None):
    """The native binding and the stream for a call whose tensors are with `t`, if that is the current device."""
    global _bound
    if _b2torch is None or not isinstance(t, torch.Tensor):
        return None, 0
    index = t.get_device()
    if index < 0 or index != torch._C._cuda_getDevice():
        return None, 0
    if _bound is None or _bound is not _lib._LIB:
        lib = _lib.load()
        _b2torch.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in
                        ("b2_kv8_decode_step", "b2_kv8_append", "b2_kv8_prefill_attn", "b2_tables_extend")))
        _bound = lib
    return _b2torch, torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream


_I32, _F32, _BF16, _E4M3 = torch.int32, torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _is(t: torch.Tensor, name: str, dtype: torch.dtype, like: torch.Tensor, index: int, shape: tuple) -> int:
    """Address of a contiguous tensor of this type and shape on like's device (index `index`)."""
    if t.__class__ is torch.Tensor and t.dtype is dtype and t.get_device() == index and t.shape == shape and \
            t.is_contiguous():
        return t.data_ptr()
    _need(t, name, dtype, like.device, shape)      # (a parameter or another subclass passes here)
    return t.data_ptr()


def _launch(call: str, index: int, stream: torch.cuda.Stream | None, *args) -> None:
    """One library call on the device with this index, which is made current for it, on `stream` or the
    device's current one."""
    if index < 0:
        raise ValueError(f"{call}: tensors must be on a CUDA device")
    fn = getattr(_lib.load(), call)
    raw = torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, raw)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, raw)
    if rc:
        _lib.check(rc, call)


def _need_cache(k_pool, v_pool, k_scale, v_scale, like: torch.Tensor, index: int) -> tuple:
    """Addresses of the pools and scales, and the number of blocks."""
    blocks = k_pool.shape[0] if isinstance(k_pool, torch.Tensor) and k_pool.dim() == 4 else 0
    return (_is(k_pool, "k_pool", _E4M3, like, index, (blocks, HKV, BLOCK, D)),
            _is(v_pool, "v_pool", _E4M3, like, index, (blocks, HKV, D, BLOCK)),
            _is(k_scale, "k_scale", _F32, like, index, (blocks, HKV)),
            _is(v_scale, "v_scale", _F32, like, index, (blocks, HKV)), blocks)


def _need_tables(block_tables, past_lens, chunk_lens, like: torch.Tensor, index: int) -> tuple:
    """Batch, table width, and the addresses of tables, past and chunk lengths."""
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be [batch, max_blocks_per_seq]")
    b, width = block_tables.shape
    return (b, width, _is(block_tables, "block_tables", _I32, like, index, (b, width)),
            _is(past_lens, "past_lens", _I32, like, index, (b,)),
            None if chunk_lens is None else _is(chunk_lens, "chunk_lens", _I32, like, index, (b,)))


def _need_qk(mode: int, gamma_q, gamma_k, eps: float, cos, sin, like: torch.Tensor, index: int) -> tuple:
    """The q/k norm and RoPE arguments of a call."""
    gq = gk = c = s = None
    rows = 0
    if mode & _lib.B2_NORM_QK:
        gq = _is(gamma_q, "gamma_q", _BF16, like, index, (D,))
        gk = _is(gamma_k, "gamma_k", _BF16, like, index, (D,))
    if mode & _lib.B2_ROPE_QK:
        rows = _need_rope(cos, sin, like.device)
        c, s = cos.data_ptr(), sin.data_ptr()
    return gq, gk, eps, c, s, rows


def _need_err(dev_err, like: torch.Tensor, index: int) -> int:
    return _is(dev_err, "dev_err", _I32, like, index, (1,))


def _need_workspace(workspace, like: torch.Tensor, index: int) -> tuple:
    if not isinstance(workspace, torch.Tensor) or workspace.dtype is not torch.uint8 or \
            workspace.get_device() != index or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {like.device} (workspace_kv8)")
    return workspace.data_ptr(), workspace.numel()


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
    RoPE) as the table builder writes them, a negative slot skipping its row
    (rows of one block follow one another, at consecutive slots and without
    skipped rows between them; later ones are refused in dev_err);
    or [batch, tokens, >= 2048] with past_lens and block_tables.  q_out: bf16
    [rows, 16, 64] normalised and rotated query."""
    if not isinstance(qkv, torch.Tensor) or qkv.dim() not in (2, 3) or qkv.shape[-1] < QKV_WIDTH:
        raise ValueError(f"qkv must be [rows or batch x tokens, >= {QKV_WIDTH}]")
    index, shape = qkv.get_device(), qkv.shape
    width = shape[-1]
    rows = qkv.numel() // width
    q = _is(qkv, "qkv", _BF16, qkv, index, shape)
    tokens = table_width = 0
    slot = place = past = chunk = tables = None
    if slots is not None:
        slot = _is(slots, "slots", _I32, qkv, index, (rows,))
        if positions is not None:
            place = _is(positions, "positions", _I32, qkv, index, (rows,))
    else:
        if len(shape) != 3:
            raise ValueError("without slots, qkv must be [batch, tokens, width]")
        b, table_width, tables, past, chunk = _need_tables(block_tables, past_lens, chunk_lens, qkv, index)
        tokens = shape[1]
        if b != shape[0]:
            raise ValueError(f"block_tables must have {shape[0]} rows, got {b}")
    cache = _need_cache(k_pool, v_pool, k_scale, v_scale, qkv, index) \
        if mode & _lib.B2_STORE_KV or slots is not None else (None, None, None, None, 0)
    q_to = None if q_out is None else _is(q_out, "q_out", _BF16, qkv, index, (rows, HQ, D))
    _launch("b2_kv8_append", index, stream, q, width, rows, slot, place, past, chunk, tokens, tables, table_width,
            *_need_qk(mode, gamma_q, gamma_k, eps, cos, sin, qkv, index), *cache, q_to, mode,
            _need_err(dev_err, qkv, index))


def decode_step_kv8(qkv: torch.Tensor, past_lens: torch.Tensor, *, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor, out: torch.Tensor,
                    workspace: torch.Tensor, dev_err: torch.Tensor, chunk_lens: torch.Tensor | None = None,
                    gamma_q: torch.Tensor | None = None, gamma_k: torch.Tensor | None = None,
                    cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, mode: int = NORM_ROPE_STORE,
                    eps: float = EPS, scale: float = SCALE, stream: torch.cuda.Stream | None = None,
                    row_start: torch.Tensor | None = None, max_tokens: int | None = None) -> None:
    """One decode step over the 8-bit cache (b2_kv8_decode_step): raw
    projections of up to 4 new tokens per sequence at positions past_lens[b] + t.

    Padded: qkv bf16 [B, T, >= 2048], T of 1 to 4, chunk_lens[b] (0 to T; None:
    T) of them there.
    Packed: qkv bf16 [rows, >= 2048], sequence b's chunk_lens[b] <= max_tokens
    tokens (None: max_tokens) from row row_start[b] on.

    Appends their k/v and writes the contexts into out ([B, T, 16, 64], packed
    [rows, 16, 64]); rows of no token stay as they were.  The sequences' last
    blocks are distinct: no two entries append to one sequence.  `mode` as
    decode_step's."""
    native, raw = _native(qkv, stream)
    if native is not None:
        rc = native.step(qkv, past_lens, k_pool, v_pool, k_scale, v_scale, block_tables, out, workspace, dev_err,
                         chunk_lens, gamma_q, gamma_k, cos, sin, mode, eps, scale, raw, row_start, max_tokens)
        if rc == 0:
            return
        if rc is not None:
            _lib.check(rc, "b2_kv8_decode_step")
    if not isinstance(qkv, torch.Tensor) or qkv.dim() not in (2, 3) or qkv.shape[-1] < QKV_WIDTH:
        raise ValueError(f"qkv must be [rows, >= {QKV_WIDTH}] or [batch, tokens, >= {QKV_WIDTH}]")
    padded, width = qkv.dim() == 3, qkv.shape[-1]
    if padded != (row_start is None) or padded != (max_tokens is None):
        raise ValueError("packed qkv [rows, width] needs row_start and max_tokens, padded qkv neither")
    t = qkv.shape[1] if padded else int(max_tokens)
    if not 1 <= t <= MAX_STEP_TOKENS:
        raise ValueError(f"tokens must be in [1, {MAX_STEP_TOKENS}], got {t}")
    index = qkv.get_device()
    q = _is(qkv, "qkv", _BF16, qkv, index, qkv.shape)
    b, table_width, tables, past, chunk = _need_tables(block_tables, past_lens, chunk_lens, qkv, index)
    if padded and b != qkv.shape[0]:
        raise ValueError(f"block_tables must have {qkv.shape[0]} rows, got {b}")
    rows = b * t if padded else qkv.shape[0]
    start = None if padded else _is(row_start, "row_start", _I32, qkv, index, (b,))
    _launch("b2_kv8_decode_step", index, stream, q, width, rows, start, t, chunk,
            *_need_qk(mode, gamma_q, gamma_k, eps, cos, sin, qkv, index), past, tables, table_width,
            *_need_cache(k_pool, v_pool, k_scale, v_scale, qkv, index), b, scale, mode,
            _is(out, "out", _BF16, qkv, index, (*qkv.shape[:-1], HQ, D)), *_need_workspace(workspace, qkv, index),
            _need_err(dev_err, qkv, index))


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
    native, raw = _native(qkv, stream) if out is not None else (None, 0)
    if native is not None and qkv.dim() >= 2 and qkv.shape[-1] >= QKV_WIDTH:
        q_buf = None
        if mode & (_lib.B2_NORM_QK | _lib.B2_ROPE_QK):
            with torch.cuda.stream(stream):     # freed behind the kernels that use it
                q_buf = torch.empty(qkv.numel() // qkv.shape[-1], HQ, D, dtype=_BF16, device=qkv.device)
        rc = native.prefill(qkv, past_lens, k_pool, v_pool, k_scale, v_scale, block_tables, out, workspace, dev_err,
                            chunk_lens, gamma_q, gamma_k, cos, sin, mode, eps, scale, raw, row_start, max_tokens, slots,
                            positions, q_buf)
        if rc == 0:
            return out
        if rc is not None:
            _lib.check(rc, "b2_kv8_append / b2_kv8_prefill_attn")
    if not isinstance(qkv, torch.Tensor) or qkv.dim() not in (2, 3) or qkv.shape[-1] < QKV_WIDTH:
        raise ValueError(f"qkv must be [rows, >= {QKV_WIDTH}] or [batch, tokens, >= {QKV_WIDTH}]")
    index = qkv.get_device()
    width = qkv.shape[-1]
    rows = qkv.numel() // width
    b, table_width, tables, past, chunk = _need_tables(block_tables, past_lens, chunk_lens, qkv, index)
    start = None
    if qkv.dim() == 3:
        tokens = qkv.shape[1]
        if qkv.shape[0] != b or row_start is not None:
            raise ValueError(f"padded qkv must be [{b}, tokens, width], without row_start")
        shape = (b, tokens, HQ, D)
    else:
        if row_start is None or max_tokens is None or slots is None:
            raise ValueError("packed qkv needs row_start, max_tokens and slots")
        start = _is(row_start, "row_start", _I32, qkv, index, (b,))
        tokens = int(max_tokens)
        shape = (rows, HQ, D)
    if out is None:
        with torch.cuda.stream(stream):
            out = torch.zeros(shape, dtype=_BF16, device=qkv.device)
    to = _is(out, "out", _BF16, qkv, index, shape)
    cache = _need_cache(k_pool, v_pool, k_scale, v_scale, qkv, index)
    work = _need_workspace(workspace, qkv, index)
    err = _need_err(dev_err, qkv, index)
    q = _is(qkv, "qkv", _BF16, qkv, index, qkv.shape)
    slot = None if slots is None else _is(slots, "slots", _I32, qkv, index, (rows,))
    place = None if positions is None else _is(positions, "positions", _I32, qkv, index, (rows,))
    qk = _need_qk(mode, gamma_q, gamma_k, eps, cos, sin, qkv, index)
    turned = mode & (_lib.B2_NORM_QK | _lib.B2_ROPE_QK)
    with torch.cuda.stream(stream):
        q_buf = torch.empty(rows, HQ, D, dtype=_BF16, device=qkv.device) if turned else None
    if mode:
        _launch("b2_kv8_append", index, stream, q, width, rows, slot, place, past, chunk, tokens, tables, table_width,
                *qk, *cache, None if q_buf is None else q_buf.data_ptr(), mode, err)
    _launch("b2_kv8_prefill_attn", index, stream, q if q_buf is None else q_buf.data_ptr(),
            width if q_buf is None else HQ * D, rows, start, past, chunk, tokens, tables, table_width, *cache, b, scale,
            to, *work, err)
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
             chunk_lens: torch.Tensor | None = None, row_start: torch.Tensor | None = None,
             max_tokens: int | None = None, out: torch.Tensor | None = None,
             stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """qkv bf16 [B, W] (one token per sequence), [B, T, W] or, with row_start
        and max_tokens, packed [rows, W] raw projections; returns the contexts
        [B, 16, 64], [B, T, 16, 64] or [rows, 16, 64]."""
        if row_start is not None or max_tokens is not None:
            if out is None:
                if qkv.shape[0] > self.out.shape[0]:
                    raise ValueError(f"{qkv.shape[0]} rows > max_batch x max_tokens {self.out.shape[0]}")
                out = self.out[:qkv.shape[0]]
            decode_step_kv8(qkv, past_lens, block_tables=block_tables, chunk_lens=chunk_lens, row_start=row_start,
                            max_tokens=max_tokens, out=out, stream=stream, **self._common(layer))
            return out
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
