"""Plain restatement in 64 bits, on the CPU, of the 8-bit paged cache (codes,
scales, append), of attention over it and of the device block tables.  Test
infrastructure: loops over sequences, blocks and heads, no code of the package.
"""
import math

import torch

HQ, HKV, D, BLOCK = 16, 8, 64, 64
BIG = torch.finfo(torch.bfloat16).max


class Cache:
    """CPU copy of one layer: k codes [blocks, 8, token, dim], v codes [blocks, 8, dim, token], scales [blocks, 8]."""

    def __init__(self, k, v, ks, vs):
        self.k, self.v = k.cpu().clone(), v.cpu().clone()
        self.ks, self.vs = ks.cpu().clone(), vs.cpu().clone()

    @classmethod
    def of(cls, kw):
        return cls(kw["k_pool"], kw["v_pool"], kw["k_scale"], kw["v_scale"])

    def same_as(self, kw):
        return all(torch.equal(a.view(torch.uint8), b.cpu().view(torch.uint8))
                   for a, b in ((self.k, kw["k_pool"]), (self.v, kw["v_pool"]))) and \
            torch.equal(self.ks.view(torch.int32), kw["k_scale"].cpu().view(torch.int32)) and \
            torch.equal(self.vs.view(torch.int32), kw["v_scale"].cpu().view(torch.int32))


def scale_of(amax: float) -> float:
    """Smallest power of two s >= 2^-100 with amax <= 448 s."""
    e = -100
    if amax > 0:
        e = max(e, math.frexp(amax)[1] - 10)        # 448 * 2^(e) is above amax / 4 here: step up to it
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return 2.0 ** e


def encode(x, s):
    return (x.clamp(-BIG, BIG).double() / s).clamp(-448, 448).float().to(torch.float8_e4m3fn)


def append(c: Cache, table, past: int, k, v) -> None:
    """k, v bf16 [n, 8, 64] at positions past .. past + n - 1 of the sequence with block table `table`."""
    n = k.shape[0]
    pos = past
    while pos < past + n:
        blk, r0 = int(table[pos // BLOCK]), pos % BLOCK
        m = min(BLOCK - r0, past + n - pos)
        for h in range(HKV):
            for x, codes, scales, dim_major in ((k, c.k, c.ks, False), (v, c.v, c.vs, True)):
                rows = x[pos - past:pos - past + m, h].float()
                mag = rows.abs().clamp(max=BIG)
                amax = float(mag[~mag.isnan()].max()) if bool((~mag.isnan()).any()) else 0.0
                old = float(scales[blk, h]) if r0 else 0.0
                s = max(scale_of(amax), old)
                tile = codes[blk, h].T if dim_major else codes[blk, h]      # [token, dim] view
                if r0 and s > old:
                    tile.view(torch.uint8)[:r0] = encode(tile[:r0].float(), s / old).view(torch.uint8)
                tile.view(torch.uint8)[r0:r0 + m] = encode(rows, s).view(torch.uint8)
                scales[blk, h] = s
        pos += m


def values(c: Cache, table, n: int):
    """K and V [8, n, 64] in 64 bits."""
    ids = [int(i) for i in table[:(n + BLOCK - 1) // BLOCK]]
    k = (c.k[ids].double() * c.ks[ids].double()[..., None, None]).transpose(0, 1).reshape(HKV, -1, D)[:, :n]
    v = (c.v[ids].double() * c.vs[ids].double()[..., None, None]).mT.transpose(0, 1).reshape(HKV, -1, D)[:, :n]
    return k, v


def attend(c: Cache, table, past: int, q, scale=D ** -0.5):
    """q bf16 [n, 16, 64] of the tokens at past ..; the context [n, 16, 64], the weighted mean of |v| and what weights
    below the f16 range may cost (see check_context), in 64 bits."""
    n = q.shape[0]
    k, v = values(c, table, past + n)
    p = torch.einsum("thgd,hld->hgtl", q.double().view(n, HKV, 2, D), k) * scale
    hide = torch.arange(past + n)[None] > past + torch.arange(n)[:, None]
    p = torch.softmax(p.masked_fill(hide, -torch.inf), -1)
    out = torch.einsum("hgtl,hld->thgd", p, v).reshape(n, HQ, D)
    mean = torch.einsum("hgtl,hld->thgd", p, v.abs()).reshape(n, HQ, D)
    ids = [int(i) for i in table[:(past + n + BLOCK - 1) // BLOCK]]
    s = c.vs[ids].double().T.repeat_interleave(BLOCK, 1)[:, :past + n]          # scale of each token's block
    sees = (~hide).double()
    codes = torch.einsum("tl,hld->htd", sees, v.abs() / s[..., None])
    low = 2.0 ** -25 * torch.einsum("hgt,htd->thgd", (p * s[:, None, None]).amax(-1), codes).reshape(n, HQ, D)
    return out, mean, low


def check_context(got, want, mean, low, what=""):
    """The kernels' error: the bf16 result is off by half a step, 2^-8 of its
    value.  Each weight p is rounded to f16 (2^-11), its score to fp32 over 64
    products (below 2^-13 for the scores here) and its exponential by 2^-22;
    what falls below the f16 range of a 4096-token range adds 2^-13: together
    below 2^-10 in the sum and in the normaliser, so 2^-9 of the weighted mean
    of |v|.  The 2^-13 does not hold where the values of a dim are 0 but for
    tokens of small weight, all of which then falls below the range.  Exactly: a
    token's stored weight is x_j = p_j s_j / X with X <= max_j p_j s_j (s_j the
    scale of V's block), rounded with an error of at most 2^-25 below 2^-14; it
    multiplies the code v_j / s_j, and the products' sum X, so such weights cost
    at most low = 2^-25 max_j (p_j s_j) sum_j |v_j| / s_j over the visible j."""
    got, bound = got.cpu().double(), 2.0 ** -8 * want.abs() + 2.0 ** -9 * mean + low
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{what}: off by up to {float((off / bound.clamp(min=1e-30)).max()):.2f} bounds"


def split(rows):
    """qkv rows [n, >= 2048] -> q [n, 16, 64], k, v [n, 8, 64]."""
    n = rows.shape[0]
    return (rows[:, :HQ * D].reshape(n, HQ, D), rows[:, HQ * D:(HQ + HKV) * D].reshape(n, HKV, D),
            rows[:, (HQ + HKV) * D:(HQ + 2 * HKV) * D].reshape(n, HKV, D))


def extend(tables, held, free_list, count, past, new, rows, tokens_per_seq):
    """b2_tables_extend on Python lists; returns its outputs, with whether a length was bad."""
    b, width = len(tables), len(tables[0]) if tables else 0
    tables = [list(t) for t in tables]
    held, need_before, bad_any, start = list(held), 0, False, 0
    granted, starts = [], []
    slots, positions = [-1] * rows, [0] * rows
    popped = 0
    for i in range(b):
        first = i * tokens_per_seq if tokens_per_seq else start
        n = max(new[i], 0)
        bad = past[i] < 0 or new[i] < 0 or held[i] < 0 or held[i] > width or past[i] + new[i] > width * BLOCK
        bad = bad or (tokens_per_seq > 0 and new[i] > tokens_per_seq)
        if not tokens_per_seq:
            bad = bad or (n > 0 and first + n > rows)
            start += n
        need = 0 if bad else max(0, -(-(past[i] + new[i]) // BLOCK) - held[i])
        need_before += need
        ok = not bad and (need == 0 or need_before <= count)
        if ok:
            for _ in range(need):
                tables[i][held[i]] = free_list[count - 1 - popped]
                held[i] += 1
                popped += 1
        granted.append(new[i] if ok else 0)
        starts.append(min(first, rows))
        bad_any = bad_any or bad
        for t in range(n):
            r = first + t
            if r >= rows or (tokens_per_seq and t >= tokens_per_seq):
                break
            pos = past[i] + t
            positions[r] = pos
            if ok:
                slots[r] = tables[i][pos // BLOCK] * BLOCK + pos % BLOCK
    return {"tables": tables, "held": held, "count": count - popped, "granted": granted, "row_start": starts,
            "slots": slots, "positions": positions, "bad": bad_any}
