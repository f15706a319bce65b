"""What is measured of the 8-bit paged cache: the decode step and the prompt chunk over it, and the block
tables and slot maps built on the GPU.  Plain forms (own = False) and the framework's calls (own = True).

The cache, per attention layer (64-token blocks, 8 KV heads, head_dim 64, 16 query heads):
  k_pool   float8_e4m3fn [blocks][8][64 tokens][64 dims]     k_scale  float32 [blocks][8]
  v_pool   float8_e4m3fn [blocks][8][64 dims][64 tokens]     v_scale  float32 [blocks][8]
A stored code stands for code * scale of its (block, head).  Scales are powers of two: the smallest with
448 * scale >= |x| for every value in the block (never below 2^-100).  New tokens that need a larger scale
raise it, and the codes that the block already held are rounded again at the new one.
"""
import importlib
import math

import torch

own = False

HQ, HKV, D, BLOCK = 16, 8, 64, 64
WIDTH = (HQ + 2 * HKV) * D
MIN_EXP = -100      # the smallest scale is 2^MIN_EXP
BF16_MAX = 3.3895313892515355e38
PKG = "ryzenai-npu-lab_b200"


def _pkg(name):
    return importlib.import_module(PKG + "." + name)


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one chat at its start: the shortest call, latency alone
        {"name": "step_one", "op": "step", "batch": 1, "tokens": 1, "min_len": 37, "max_len": 37, "ragged": False},
        # the batched-decode benchmark: 64 sequences, lengths uniform in [128, 8192], one token each
        {"name": "step_batch", "op": "step", "batch": 64, "tokens": 1, "min_len": 128, "max_len": 8192,
         "ragged": False},
        # one long document: the 131 072-token sequence of the long-context benchmark
        {"name": "step_long", "op": "step", "batch": 1, "tokens": 1, "min_len": 131071, "max_len": 131071,
         "ragged": False},
        # a serving batch of many short answers (256 sequences of 32 to 288 tokens)
        {"name": "step_short", "op": "step", "batch": 256, "tokens": 1, "min_len": 32, "max_len": 288,
         "ragged": False},
        # drafted tokens being verified: up to 4 per sequence, some sequences with fewer or none
        {"name": "step_draft", "op": "step", "batch": 33, "tokens": 4, "min_len": 0, "max_len": 6001,
         "ragged": True},
        # a first message of 21 tokens into an empty cache
        {"name": "prompt_first", "op": "prompt", "batch": 1, "tokens": 21, "min_len": 0, "max_len": 0,
         "ragged": False, "packed": False},
        # the batched-prompt benchmark: 64 sequences, 128 new tokens over 128 to 8192 cached ones
        {"name": "prompt_batch", "op": "prompt", "batch": 64, "tokens": 128, "min_len": 128, "max_len": 8064,
         "ragged": False, "packed": False},
        # prompts of different lengths packed behind one another, some over a cached prefix
        {"name": "prompt_packed", "op": "prompt", "batch": 7, "tokens": 1999, "min_len": 0, "max_len": 777,
         "ragged": True, "packed": True},
        # the tables of one decode step of the benchmark's batch
        {"name": "tables_step", "op": "tables", "batch": 64, "min_new": 1, "max_new": 1, "min_len": 128,
         "max_len": 8191, "packed": False, "tight": False},
        # a scheduler's mixed batch: decode tokens and prompt chunks, with a pool that runs out on the way
        {"name": "tables_mixed", "op": "tables", "batch": 1001, "min_new": 0, "max_new": 97, "min_len": 0,
         "max_len": 2000, "packed": True, "tight": True},
        # admission of a large queue: a million prompt tokens at once
        {"name": "tables_queue", "op": "tables", "batch": 4096, "min_new": 1, "max_new": 511, "min_len": 0,
         "max_len": 64, "packed": True, "tight": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "step", "prompt", "tables"])
    if op == "step":
        batch = _log(rng, 1, 512)
        hi = _log(rng, 1, min(131071, 400000 // batch))
        return {"op": op, "batch": batch, "tokens": rng.choice([1, 1, 2, 3, 4]), "min_len": rng.randint(0, hi),
                "max_len": hi, "ragged": rng.random() < 0.4}
    if op == "prompt":
        tokens = _log(rng, 1, 2047)
        batch = _log(rng, 1, max(1, min(64, 8192 // tokens)))
        hi = _log(rng, 1, max(1, min(16000, 400000 // batch, 32000000 // (batch * tokens))))
        hi = rng.choice([0, hi, hi])
        return {"op": op, "batch": batch, "tokens": tokens, "min_len": rng.randint(0, hi), "max_len": hi,
                "ragged": rng.random() < 0.5, "packed": rng.random() < 0.5}
    batch = _log(rng, 1, 4096)
    hi = _log(rng, 1, max(1, min(2047, 1000000 // batch)))
    return {"op": op, "batch": batch, "min_new": rng.randint(0, hi), "max_new": hi, "min_len": 0,
            "max_len": _log(rng, 1, 4096), "packed": rng.random() < 0.5, "tight": rng.random() < 0.3}


# ------------------------------------------------------------------ inputs

def _pow2_scale(amax):
    """The smallest power of two s >= 2^MIN_EXP with amax <= 448 * s (amax >= 0, finite)."""
    m, e = torch.frexp(amax / 448.0)                # amax / 448 = m * 2^e, m in [1/2, 1)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _codes(x):
    """x as float8_e4m3fn, nearest even, limited to +-448."""
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _pool(blocks, g, dev, sigma):
    """Codes and scales of `blocks` random blocks of tiles [8][64][64]."""
    code = torch.empty(blocks, HKV, BLOCK, D, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(blocks, HKV, dtype=torch.float32, device=dev)
    for i in range(0, blocks, 2048):
        n = min(2048, blocks - i)
        x = torch.randn(n, HKV, BLOCK, D, generator=g, device=dev) * sigma
        x *= torch.exp(0.5 * torch.randn(n, HKV, 1, 1, generator=g, device=dev))     # heads and blocks differ
        s = _pow2_scale(x.abs().amax((2, 3)))
        code[i:i + n] = _codes(x / s[:, :, None, None])
        scale[i:i + n] = s
    return code, scale


def _lengths(case, g, dev, lo, hi):
    return torch.randint(case[lo], case[hi] + 1, (case["batch"],), generator=g, device=dev, dtype=torch.int32)


def _shares(n, lo, hi, g, dev):
    """n whole numbers in [lo, hi], uniform in pairs that add up to lo + hi: every seed gives the same sum."""
    x = torch.randint(lo, hi + 1, (n // 2,), generator=g, device=dev)
    x = torch.cat([x, lo + hi - x, torch.full((n % 2,), (lo + hi) // 2, device=dev)])
    return x[torch.randperm(n, generator=g, device=dev)].to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    return _prepare_tables(case, g, dev) if case["op"] == "tables" else _prepare_attention(case, g, dev)


def _prepare_attention(case, g, dev):
    b, t = case["batch"], case["tokens"]
    past = _lengths(case, g, dev, "min_len", "max_len")
    chunk = None
    if case["ragged"]:
        # a few sequences wait (no token); the first has its full share
        chunk = torch.cat([torch.full((1,), t, dtype=torch.int32, device=dev),
                           _shares(b - 1, 0 if t <= 4 else 1, t, g, dev)])
    width = (case["max_len"] + t + BLOCK - 1) // BLOCK
    need = (past.long() + t + BLOCK - 1) // BLOCK
    # each sequence holds the blocks that it needs, scattered over the pool; the last block belongs to nobody
    total = b * width if b * width <= 16384 else int(need.sum())
    blocks = total + 1
    order = torch.randperm(total, generator=g, device=dev, dtype=torch.int64)
    col = torch.arange(width, device=dev)[None]
    at = (need.cumsum(0) - need)[:, None] + col
    tables = torch.where(col < need[:, None], order[at.clamp(max=total - 1)], -1).to(torch.int32)
    k, ks = _pool(blocks, g, dev, 1.0)
    v, vs = _pool(blocks, g, dev, 0.6)
    packed = case.get("packed", False)
    if packed:
        lens = chunk if chunk is not None else torch.full((b,), t, dtype=torch.int32, device=dev)
        cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), lens.cumsum(0)])
        rows, start = int(cu[-1]), cu[:-1].to(torch.int32)
    else:
        rows, start = b * t, torch.arange(b, device=dev, dtype=torch.int32) * t
    qkv = (torch.randn(rows, WIDTH, generator=g, device=dev) *
           torch.exp(0.4 * torch.randn(rows, 1, generator=g, device=dev))).to(torch.bfloat16)
    state = {"op": case["op"], "batch": b, "tokens": t, "packed": packed, "past": past, "chunk": chunk, "start": start,
             "tables": tables, "k": k, "v": v, "ks": ks, "vs": vs, "qkv": qkv,
             "out": torch.zeros(rows, HQ, D, dtype=torch.bfloat16, device=dev),
             "err": torch.zeros(1, dtype=torch.int32, device=dev)}
    if case["op"] == "prompt":
        # the slot map and positions of the chunk's rows, as the table builder gives them once for all layers
        seq, off, ok = _rows(state)
        pos = past.long()[seq] + off
        blk = tables.long()[seq, (pos // BLOCK).clamp(max=width - 1)]
        state["slots"] = torch.where(ok, blk * BLOCK + pos % BLOCK, -1).to(torch.int32)
        state["positions"] = torch.where(ok, pos, 0).to(torch.int32)
    if own:
        state["work"] = _pkg("attention_kv8").workspace_kv8(dev)
    return state


def _prepare_tables(case, g, dev):
    b = case["batch"]
    past = _lengths(case, g, dev, "min_len", "max_len")
    new = _shares(b, case["min_new"], case["max_new"], g, dev)
    held = (past + BLOCK - 1) // BLOCK
    width = (case["max_len"] + case["max_new"] + BLOCK - 1) // BLOCK
    used = int(held.sum())
    grow = int(((past + new + BLOCK - 1) // BLOCK - held).sum())
    free = max(1, grow // 2) if case["tight"] else grow + 16
    order = torch.randperm(used + free, generator=g, device=dev, dtype=torch.int64)
    col = torch.arange(width, device=dev)[None]
    at = (held.long().cumsum(0) - held)[:, None] + col
    tables = torch.where(col < held[:, None], order[at.clamp(max=max(used - 1, 0))], -1).to(torch.int32)
    free_list = torch.zeros(used + free, dtype=torch.int32, device=dev)
    free_list[:free] = order[used:].to(torch.int32)
    rows = int(new.sum()) + 5 if case["packed"] else b * case["max_new"]     # packed: a buffer with some room left

    def ints(n):
        return torch.zeros(n, dtype=torch.int32, device=dev)
    return {"op": "tables", "batch": b, "packed": case["packed"], "tokens": case["max_new"], "past": past, "new": new,
            "held": held, "tables": tables, "free": free_list,
            "count": torch.full((1,), free, dtype=torch.int32, device=dev),
            "held_out": ints(b), "count_out": ints(1), "granted": ints(b), "start": ints(b), "slots": ints(rows),
            "positions": ints(rows), "err": ints(1)}


# ------------------------------------------------------------------ the operators

def run(state):
    return {"step": _run_step, "prompt": _run_prompt, "tables": _run_tables}[state["op"]](state)


def _cache(s):
    return {"out": s["out"], "k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _run_step(s):
    if not own:
        return _plain_attention(s)
    _pkg("attention_kv8").decode_step_kv8(
        s["qkv"].view(s["batch"], s["tokens"], WIDTH), s["past"], k_pool=s["k"], v_pool=s["v"], k_scale=s["ks"],
        v_scale=s["vs"], block_tables=s["tables"], chunk_lens=s["chunk"],
        out=s["out"].view(s["batch"], s["tokens"], HQ, D), workspace=s["work"], dev_err=s["err"],
        mode=_pkg("_lib").B2_STORE_KV)
    return _cache(s)


def _run_prompt(s):
    if not own:
        return _plain_attention(s)
    _pkg("attention_kv8").prefill_kv8(
        s["qkv"], s["past"], k_pool=s["k"], v_pool=s["v"], k_scale=s["ks"], v_scale=s["vs"],
        block_tables=s["tables"], row_start=s["start"], chunk_lens=s["chunk"], max_tokens=s["tokens"],
        slots=s["slots"], positions=s["positions"], out=s["out"], workspace=s["work"], dev_err=s["err"],
        mode=_pkg("_lib").B2_STORE_KV)
    return _cache(s)


def _run_tables(s):
    if not own:
        return _plain_tables(s)
    _pkg("block_tables").extend_tables(
        s["tables"], s["held"], s["free"], s["count"], s["past"], s["new"], held_out=s["held_out"],
        free_count_out=s["count_out"], granted=s["granted"], row_start=s["start"], slots=s["slots"],
        positions=s["positions"], tokens_per_seq=0 if s["packed"] else s["tokens"], dev_err=s["err"])
    return {"tables": s["tables"], "held": s["held_out"], "count": s["count_out"], "granted": s["granted"],
            "start": s["start"], "slots": s["slots"], "positions": s["positions"]}


def _rows(s):
    """Sequence, token and validity of each row of qkv."""
    n, t = s["qkv"].shape[0], s["tokens"]
    row = torch.arange(n, device=s["qkv"].device)
    seq = torch.searchsorted(s["start"].long(), row, right=True) - 1 if s["packed"] else row // t
    off = row - s["start"].long()[seq]
    return seq, off, off < (s["chunk"].long()[seq] if s["chunk"] is not None else t)


def _append(code, scale, x, blk, new, old, touched, v):
    """The touched tiles with the new tokens x [b, j, 64, 8, 64] (token-major; `v`: tiles are dim-major)."""
    tile = code.view(torch.uint8)[blk].view(torch.float8_e4m3fn).float()        # [b, j, 8, 64, 64]
    if v:
        tile = tile.transpose(-1, -2)
    x = x.permute(0, 1, 3, 2, 4).clamp(-BF16_MAX, BF16_MAX)
    m_new, m_old = new[:, :, None, :, None], old[:, :, None, :, None]
    s_old = torch.where(old.any(-1)[:, :, None], scale[blk], 0.0)
    s_new = torch.maximum(_pow2_scale(torch.where(m_new, x.abs(), 0.0).amax((3, 4))), s_old)
    ratio = (s_old / s_new)[..., None, None]
    y = torch.where(m_new, _codes(x / s_new[..., None, None]).float(),
                    torch.where(m_old & (ratio < 1), _codes(tile * ratio).float(), tile))
    if v:
        y = y.transpose(-1, -2)
    code.view(torch.uint8)[blk] = y.to(torch.float8_e4m3fn).view(torch.uint8)
    scale[blk] = torch.where(touched[:, :, None], s_new, scale[blk])


def _plain_attention(s):
    """Append the new tokens to the cache, then causal attention of each over everything cached so far."""
    b, t, past = s["batch"], s["tokens"], s["past"].long()
    dev = past.device
    chunk = s["chunk"].long() if s["chunk"] is not None else torch.full((b,), t, device=dev)
    spare = s["k"].shape[0] - 1
    tables = s["tables"].long()
    width = tables.shape[1]
    # the rows as [b, t]; a row that a sequence does not have is row 0 and masked
    tok = torch.arange(t, device=dev)[None]
    live = tok < chunk[:, None]                                                    # [b, t]
    row = torch.where(live, s["start"].long()[:, None] + tok, 0)
    x = s["qkv"][row].float()
    q = x[..., :HQ * D].reshape(b, t, HKV, HQ // HKV, D)
    k_new = x[..., HQ * D:(HQ + HKV) * D].reshape(b, t, HKV, D)
    v_new = x[..., (HQ + HKV) * D:].reshape(b, t, HKV, D)
    # append: the blocks that new tokens may touch
    j = (past // BLOCK)[:, None] + torch.arange((t + BLOCK - 1) // BLOCK + 1, device=dev)[None]
    pos = j[:, :, None] * BLOCK + torch.arange(BLOCK, device=dev)
    i = pos - past[:, None, None]
    new, old = (i >= 0) & (i < chunk[:, None, None]), i < 0
    touched = new.any(-1)
    blk = torch.where(touched, torch.gather(tables, 1, j.clamp(max=width - 1)), spare)
    old = old & touched[:, :, None]
    pick = (torch.arange(b, device=dev)[:, None, None], i.clamp(0, t - 1))
    _append(s["k"], s["ks"], k_new[pick], blk, new, old, touched, False)
    _append(s["v"], s["vs"], v_new[pick], blk, new, old, touched, True)
    # attention over the cache
    at = torch.where(tables >= 0, tables, spare)
    k = s["k"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * s["ks"][at][..., None, None]
    v = s["v"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * s["vs"][at][..., None, None]
    k = k.transpose(1, 2).reshape(b, HKV, width * BLOCK, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, HKV, width * BLOCK, D)
    key = torch.arange(width * BLOCK, device=dev)
    v = torch.where((key < (past + chunk)[:, None])[:, None, :, None], v, 0.0)
    see = key <= (past[:, None] + tok)[..., None]                                  # [b, t, keys]
    q = q.permute(0, 2, 3, 1, 4).reshape(b, HKV, -1, D)
    p = (q @ k.transpose(-1, -2) * D ** -0.5).view(b, HKV, HQ // HKV, t, -1)
    p = torch.where(see[:, None, None], p, -torch.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    o = (p.view(b, HKV, -1, width * BLOCK) @ v).view(b, HKV, HQ // HKV, t, D) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, t, HQ, D).to(torch.bfloat16)
    out = torch.cat([s["out"], s["out"][:1]])                                      # one row for those that are not there
    out[torch.where(live, row, out.shape[0] - 1)] = o
    s["out"].copy_(out[:-1])
    return _cache(s)


def _plain_tables(s):
    """The new blocks of every request off the end of the free list, and the slot of every new token."""
    past, new, held, tables = s["past"].long(), s["new"].long(), s["held"].long(), s["tables"]
    dev, n = past.device, s["slots"].shape[0]
    need = ((past + new + BLOCK - 1) // BLOCK - held).clamp(min=0)
    upto = need.cumsum(0)
    count = s["count"].long()
    ok = (need == 0) | (upto <= count)                        # in order; the first that does not fit gets nothing
    take = torch.where(ok, need, 0)
    col = torch.arange(tables.shape[1], device=dev)[None]
    nth = (upto - need)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < (held + take)[:, None])
    tables = torch.where(fresh, s["free"][(count - 1 - nth).clamp(0, s["free"].shape[0] - 1)], tables)
    if s["packed"]:
        start = new.cumsum(0) - new
    else:
        start = torch.arange(s["batch"], device=dev) * s["tokens"]
    row = torch.arange(n, device=dev)
    seq = torch.searchsorted(start + new, row, right=True) if s["packed"] else row // s["tokens"]
    seq = seq.clamp(max=s["batch"] - 1)
    off = row - start[seq]
    live = (off >= 0) & (off < new[seq])
    pos = torch.where(live, past[seq] + off, 0)
    blk = tables.long()[seq, (pos // BLOCK).clamp(max=tables.shape[1] - 1)]
    slots = torch.where(live & ok[seq], blk * BLOCK + pos % BLOCK, -1)
    return {"tables": tables, "held": (held + take).int(), "count": (count - take.sum()).int(),
            "granted": torch.where(ok, new, 0).int(), "start": start.int(), "slots": slots.int(),
            "positions": pos.int()}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    """The contexts in 64 bits, sequence by sequence (the codes and scales have no such value)."""
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    out = s["out"].double()
    for b in range(case["batch"]):
        n = case["tokens"] if s["chunk"] is None else int(s["chunk"][b])
        past = int(s["past"][b])
        if n == 0:
            continue
        r0 = int(s["start"][b])
        rows = s["qkv"][r0:r0 + n].double()
        ids = s["tables"][b, :(past + n + BLOCK - 1) // BLOCK].long()
        caches = []
        for name, lo, dim_major in (("k", HQ * D, False), ("v", (HQ + HKV) * D, True)):
            tile = s[name].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
            if dim_major:
                tile = tile.mT
            scale = s[name + "s"][ids].double()
            fresh = rows[:, lo:lo + HKV * D].view(n, HKV, D).abs()
            for j in range(past // BLOCK, len(ids)):
                first, last = max(past, j * BLOCK), min(past + n, (j + 1) * BLOCK)
                big = fresh[first - past:last - past].amax((0, 2))
                want = torch.exp2(torch.ceil(torch.log2((big / 448).clamp(min=2.0 ** MIN_EXP))))
                kept = first - j * BLOCK
                was = scale[j] if kept else torch.zeros_like(want)
                now = torch.maximum(want, was)
                if kept:
                    again = (tile[j, :, :kept] * (was / now)[:, None, None]).float()
                    tile[j, :, :kept] = again.to(torch.float8_e4m3fn).double()
                add = rows[first - past:last - past, lo:lo + HKV * D].view(-1, HKV, D).transpose(0, 1)
                add = (add / now[:, None, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
                tile[j, :, kept:kept + last - first] = add
                scale[j] = now
            whole = (tile * scale[..., None, None]).transpose(0, 1).reshape(HKV, -1, D)
            caches.append(whole[:, :past + n])
        k, v = caches
        q = rows[:, :HQ * D].view(n, HKV, HQ // HKV, D).permute(1, 2, 0, 3)
        p = torch.einsum("hgtd,hld->hgtl", q, k) / 8.0
        hide = torch.arange(past + n, device=p.device)[None] > past + torch.arange(n, device=p.device)[:, None]
        p = torch.softmax(p.masked_fill(hide, -torch.inf), -1)
        out[r0:r0 + n] = torch.einsum("hgtl,hld->thgd", p, v).reshape(n, HQ, D)
    return {"out": out, "k": None, "v": None, "k_scale": None, "v_scale": None}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    b = case["batch"]
    mean = (case["min_len"] + case["max_len"]) / 2
    if case["op"] == "tables":
        new = (case["min_new"] + case["max_new"]) / 2
        blocks = new / BLOCK * b * (0.5 if case["tight"] else 1.0)
        rows = new * b if case["packed"] else case["max_new"] * b
        # past, new, held in; held, granted, start out; slots and positions out; a free id in and an entry out
        return {"bytes": 24 * b + 8 * rows + 8 * blocks, "flops": 0}
    t = case["tokens"]
    if case["ragged"]:
        t = (t + (0 if t <= 4 else 1)) / 2
    cached = b * mean * HKV * (2 * D + 8 / BLOCK)            # codes and scales of the cached tokens
    rows = b * t * (WIDTH * 2 + HQ * D * 2 + HKV * 2 * D)     # qkv in, context out, codes out
    tables = b * (mean + t) / BLOCK * 4 + 4 * b
    return {"bytes": cached + rows + tables, "flops": 4.0 * D * HQ * b * t * (mean + (t + 1) / 2)}
