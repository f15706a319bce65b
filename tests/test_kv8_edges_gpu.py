"""The 8-bit cache and the block tables at the edges of what a call may hold: sequences that are refused whole, NaN in
places that a token does not see, weights, queries and values at the ends of their ranges."""
import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg
from test_kv8_gpu import BF16, BLOCK, I32, _build, _err, _ints, _mods, _rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ refused sequences

@pytest.mark.parametrize("call", ["append", "prefill"])
@pytest.mark.parametrize("past,chunk", [(-5, 70), (-70, 70), (-(2 ** 31), 70), ("end", 70), (2 ** 31 - 1, 70), (30, 71),
                                        (30, 2 ** 31 - 1), (30, -1)])
def test_a_refused_sequence_is_left_as_it_was(cuda, call, past, chunk):
    """A length that does not fit refuses the whole sequence: none of its rows is stored, the other's are."""
    a8, _, lib = _mods()
    cache, ref = _build([100, 30, 64], cuda, seed=201, room=200)
    tables = cache.block_tables()
    width = tables.shape[1]
    bad = width * BLOCK - 69 if past == "end" else past
    rows = _rows(3 * 70, 202, cuda, sigma=30.0).view(3, 70, 2048)      # would raise the scales
    err = _err(cuda)
    args = dict(past_lens=_ints([100, bad, 64], cuda), block_tables=tables, chunk_lens=_ints([70, chunk, 3], cuda),
                dev_err=err, mode=lib.B2_STORE_KV, **cache.kv8())
    if call == "append":
        a8.append_kv8(rows.to(cuda), **args)
    else:
        out = torch.full((3, 70, 16, 64), -7.0, dtype=BF16, device=cuda)
        a8.prefill_kv8(rows.to(cuda), out=out, workspace=a8.workspace_kv8(cuda), **args)
        assert bool((out[1] == -7.0).all()) and bool((out[2, 3:] == -7.0).all())
    assert err.item() == lib.B2_DEV_BAD_LENGTH
    for b, p, n in ((0, 100, 70), (2, 64, 3)):
        q, k, v = ora.split(rows[b, :n])
        ora.append(ref, tables[b].cpu(), p, k, v)
        if call == "prefill":
            ora.check_context(out[b, :n], *ora.attend(ref, tables[b].cpu(), p, q), f"sequence {b}")
    assert ref.same_as(cache.kv8())


def test_prefill_flags_a_negative_chunk(cuda):
    """Packed rows and a batch whose tiles are sorted, too."""
    a8, _, lib = _mods()
    for b in (2, 40):
        cache, _ = _build([30] * b, cuda, seed=203, room=80)
        rows = _rows(b * 65, 204, cuda).to(cuda)
        slots = _ints([-1] * (65 * b), cuda)
        out = torch.full((65 * b, 16, 64), -7.0, dtype=BF16, device=cuda)
        err = _err(cuda)
        a8.prefill_kv8(rows, _ints([30] * b, cuda), block_tables=cache.block_tables(), workspace=a8.workspace_kv8(cuda),
                       dev_err=err, mode=lib.B2_STORE_KV, chunk_lens=_ints([1] * (b - 1) + [-3], cuda),
                       row_start=_ints([65 * i for i in range(b)], cuda), max_tokens=65, slots=slots, out=out,
                       **cache.kv8())
        assert err.item() == lib.B2_DEV_BAD_LENGTH
        assert bool((out.view(b, 65, 16, 64)[-1] == -7.0).all())


@pytest.mark.parametrize("many", [False, True])         # one row per thread, eight
def test_slot_map_refuses_a_request_whole(cuda, many):
    """Slots of a request whose lengths do not fit are -1, all of them, as extend_tables writes them."""
    bt, lib = load_pkg("block_tables"), load_pkg("_lib")
    top = 140000 if many else 40
    width = (200 + top + 63) // 64
    tables = torch.arange(5 * width, dtype=I32, device=cuda).view(5, width)
    end = width * 64

    def run(past, new, starts, rows, tps):
        slots, positions, err = _ints([9] * rows, cuda), _ints([9] * rows, cuda), _err(cuda)
        bt.slot_map(tables, _ints(past, cuda), _ints(new, cuda), num_blocks=5 * width, slots=slots, positions=positions,
                    row_start=None if starts is None else _ints(starts, cuda), tokens_per_seq=tps, dev_err=err)
        return slots.cpu(), err.item()

    def check(past, new, starts, rows, tps, refused):
        slots, flags = run(past, new, starts, rows, tps)
        assert flags == (lib.B2_DEV_BAD_LENGTH if refused else 0)
        want = torch.full((rows,), -1, dtype=I32)
        for b in range(5):
            if b not in refused and new[b] > 0:
                at = b * tps if starts is None else starts[b]
                pos = past[b] + torch.arange(new[b])
                want[at:at + new[b]] = ((b * width + pos // 64) * 64 + pos % 64).to(I32)
        assert torch.equal(slots, want)
    good, n = [10, 64, 0, 7, 200], [top, 3, 0, 17, top]
    starts = [2, 2 + top, 9 + top, 9 + top, 30 + top]
    rows = 30 + 2 * top
    check(good, n, starts, rows, 0, ())
    check(good, n, None, 5 * top, top, ())
    for past in (-1, -(2 ** 31), end - top + 1, 2 ** 31 - 1):
        bad = [past] + good[1:]
        check(bad, n, starts, rows, 0, (0,))
        check(bad, n, None, 5 * top, top, (0,))
    check(good, [top + 1, 3, 0, 17, top], None, 5 * top, top, (0,))          # more tokens than a padded row has
    check(good, [top, 3, -4, 17, top], starts, rows, 0, (2,))
    check(good, [top, 3, -4, 17, top], None, 5 * top, top, (2,))
    check(good, n, starts, rows - 1, 0, (4,))                                # rows behind the last one
    check(good, n, [-2] + starts[1:], rows, 0, (0,))                         # before the first one


# ------------------------------------------------------------------ NaN that a token does not see

def _spoil(rows, at):
    """NaN in the V of (sequence, token, KV head, dim) and, where dim is None, in one K value of the token's head."""
    rows = rows.clone()
    for b, t, h, d in at:
        rows[b, t, (16 + h) * 64 + 5 if d is None else (24 + h) * 64 + d] = float("nan")
    return rows


def _check_nan(ref, table, past, rows, out, what):
    """NaN where a visible token's V (or a visible K) is NaN; elsewhere the context, as if every NaN were a 0."""
    q = ora.split(rows)[0]
    n = rows.shape[0]
    clean = ora.Cache(ref.k, ref.v, ref.ks, ref.vs)
    bad_k, bad_v = clean.k.float().isnan(), clean.v.float().isnan()
    clean.k.view(torch.uint8)[bad_k] = 0
    clean.v.view(torch.uint8)[bad_v] = 0
    marks = ora.Cache(ref.k, ref.v, ref.ks, ref.vs)
    marks.k, marks.v = bad_k.float(), bad_v.float()
    marks.ks, marks.vs = torch.ones_like(ref.ks), torch.ones_like(ref.vs)
    k, v = ora.values(marks, table, past + n)                                   # [8, tokens, 64], 1 where NaN
    sees = (torch.arange(past + n)[None] <= past + torch.arange(n)[:, None]).double()
    nan = torch.einsum("tl,hld->thd", sees, v) + torch.einsum("tl,hl->th", sees, k.amax(-1))[..., None] > 0
    nan = nan.repeat_interleave(2, 1)                                           # [n, 16, 64]
    got = out.cpu()
    assert torch.equal(got.isnan(), nan), what
    want, mean, low = ora.attend(clean, table, past, q)
    zero = torch.zeros((), dtype=torch.float64)
    ora.check_context(torch.where(nan, zero.to(BF16), got), *(torch.where(nan, zero, x) for x in (want, mean, low)), what)


@pytest.mark.parametrize("tokens", [2, 3, 4])
@pytest.mark.parametrize("store", [True, False])
def test_step_nan_of_a_later_token(cuda, tokens, store):
    """A drafted token's NaN stays out of the tokens in front of it, across the edge of a block, too."""
    a8, _, lib = _mods()
    lens = [0, 61, 62, 63, 64, 200, 2000]
    cache, ref = _build([n + (0 if store else tokens) for n in lens], cuda, seed=211, room=8)
    tables = cache.block_tables()
    rows = _rows(len(lens) * tokens, 212, cuda).view(len(lens), tokens, 2048)
    last = tokens - 1
    at = [(b, t, (b + t) % 8, (7 * b + 11 * t) % 64) for b in range(len(lens)) for t in range(1, tokens)]
    at += [(1, last, 2, d) for d in range(64)] + [(3, last, 4, None), (5, last, 0, None), (5, 0, 6, 13), (6, last, 7, 63)]
    rows = _spoil(rows, at)
    if not store:       # the tokens are in the cache already
        a8.append_kv8(rows.to(cuda), past_lens=_ints(lens, cuda), block_tables=tables, dev_err=_err(cuda),
                      mode=lib.B2_STORE_KV, **cache.kv8())
    out = torch.zeros(len(lens), tokens, 16, 64, dtype=BF16, device=cuda)
    err = _err(cuda)
    a8.decode_step_kv8(rows.to(cuda), _ints(lens, cuda), block_tables=tables, out=out, workspace=a8.workspace_kv8(cuda),
                       dev_err=err, mode=lib.B2_STORE_KV if store else 0, **cache.kv8())
    assert err.item() == 0
    for b, p in enumerate(lens):
        _, k, v = ora.split(rows[b])
        ora.append(ref, tables[b].cpu(), p, k, v)
    for b, p in enumerate(lens):
        _check_nan(ref, tables[b].cpu(), p, rows[b], out[b], f"sequence {b}")


@pytest.mark.parametrize("lens,tokens", [([0], 64), ([0, 37, 64], 130), ([5000], 70), ([1, 300] * 20, 65)])
def test_prefill_nan_of_a_later_token(cuda, lens, tokens):
    """The same for a chunk: one tile, several, keys split over CTAs, tiles sorted."""
    a8, _, lib = _mods()
    cache, ref = _build(lens, cuda, seed=213, room=tokens + 3)
    tables = cache.block_tables()
    rows = _rows(len(lens) * tokens, 214, cuda).view(len(lens), tokens, 2048)
    at = []
    for b in range(min(len(lens), 4)):
        at += [(b, t, (b + t) % 8, (5 * t) % 64) for t in (0, 1, 17, 40, 62, 63)]
        at += [(b, tokens - 1, 3, d) for d in range(64)] + [(b, tokens - 2, 5, None)]
    rows = _spoil(rows, at)
    out = torch.zeros(len(lens), tokens, 16, 64, dtype=BF16, device=cuda)
    err = _err(cuda)
    a8.prefill_kv8(rows.to(cuda), _ints(lens, cuda), block_tables=tables, out=out, workspace=a8.workspace_kv8(cuda),
                   dev_err=err, mode=lib.B2_STORE_KV, **cache.kv8())
    assert err.item() == 0
    for b in range(min(len(lens), 6)):
        _, k, v = ora.split(rows[b])
        ora.append(ref, tables[b].cpu(), lens[b], k, v)
        _check_nan(ref, tables[b].cpu(), lens[b], rows[b], out[b], f"sequence {b}")


# ------------------------------------------------------------------ the ends of the ranges

def _line(cuda, k0, v, room=8):
    """One sequence whose keys are k0[j] in dim 0 and 0 elsewhere, with values v [8, n, 64]."""
    _, pc, _ = _mods()
    n = k0.numel()
    cache = pc.PagedKVCache8(pc.blocks_for(n + room) + 1, n + room, device=cuda, fill=float("nan"))
    cache.add_sequence(n)
    k = torch.zeros(8, n, 64)
    k[:, :, 0] = k0
    cache.write_dense(0, 0, k.to(BF16), v.to(BF16))
    return cache, ora.Cache.of(cache.kv8())


def _contexts(cuda, cache, rows, past, prefill):
    a8, _, lib = _mods()
    t = rows.shape[0]
    out = torch.zeros(1, t, 16, 64, dtype=BF16, device=cuda)
    err = _err(cuda)
    (a8.prefill_kv8 if prefill else a8.decode_step_kv8)(
        rows[None].to(cuda), _ints([past], cuda), block_tables=cache.block_tables(), out=out,
        workspace=a8.workspace_kv8(cuda), dev_err=err, mode=lib.B2_STORE_KV, **cache.kv8())
    assert err.item() == 0
    return out[0].cpu()


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("n", [500, 5000, 30000])
def test_many_small_weights_beside_a_large_one(cuda, prefill, n):
    """A token that takes the weight and has no value, and a flat tail at 2^-26 of it: the tail is the context.

    A weight's f16 form is at least 2^-33 of the largest product, so rounding it costs at most 2^-33 of that per
    unit of the code it multiplies: 2^-8 of check_context's `low`, which allows 2^-25."""
    k0 = torch.full((n,), -2.0)
    k0[0] = 16.0                                        # 18 nats above the others
    g = torch.Generator().manual_seed(n)
    v = 1.0 + 0.25 * torch.randn(8, n, 64, generator=g)
    v[:, 0] = 0
    cache, ref = _line(cuda, k0, v, room=40)
    t = 33 if prefill else 3
    rows = _rows(t, 221, cuda)
    rows[:, :1024] = 0
    rows[:, :1024:64] = 8.0                             # a query's score is its key's dim 0
    rows[:, 1024:1536] = 0
    rows[:, 1024:1536:64] = -2.0
    out = _contexts(cuda, cache, rows, n, prefill)
    table = cache.block_tables()[0].cpu()
    q, k, val = ora.split(rows)
    ora.append(ref, table, n, k, val)
    want, mean, low = ora.attend(ref, table, n, q)
    ora.check_context(out, want, mean, low * 2.0 ** -8)


@pytest.mark.parametrize("prefill", [False, True])
def test_query_values_far_apart(cuda, prefill):
    """A query with one value 2^27 times the others, where every key is 0: the others decide."""
    _, pc, _ = _mods()
    lens = [3, 6, 9, 17]
    for n in lens:
        g = torch.Generator().manual_seed(n)
        cache = pc.PagedKVCache8(3, 128, device=cuda, fill=float("nan"))
        cache.add_sequence(n)
        k = 2.0 * torch.randn(8, n, 64, generator=g)
        k[:, :, 3] = 0
        cache.write_dense(0, 0, k.to(BF16), torch.randn(8, n, 64, generator=g).to(BF16))
        ref = ora.Cache.of(cache.kv8())
        rows = _rows(6 if prefill else 4, 231 + n, cuda)
        rows[:, 3:1024:64] = 2.0 ** 27
        rows[:, 1024 + 3:1536:64] = 0
        out = _contexts(cuda, cache, rows, n, prefill)
        table = cache.block_tables()[0].cpu()
        q, k, v = ora.split(rows)
        ora.append(ref, table, n, k, v)
        ora.check_context(out, *ora.attend(ref, table, n, q), f"{n} tokens")


@pytest.mark.parametrize("prefill", [False, True])
def test_huge_values_of_no_weight_behind_zeros(cuda, prefill):
    """Values of 1e30 whose weight is 2^-230, in turn with blocks of zeros that have all the weight: no weight of 0
    may meet a factor that left fp32."""
    n = 64 * 600
    even = torch.arange(n) // BLOCK % 2 == 0
    k0 = torch.where(even, 10.0, -10.0)
    v = 1e30 * torch.randn(8, n, 64, generator=torch.Generator().manual_seed(1))
    v[:, even] = 0
    cache, _ = _line(cuda, k0, v)
    rows = torch.zeros(4, 2048, dtype=BF16)
    rows[:, :1024:64] = 64.0
    rows[:, 1024:1536:64] = -10.0
    out = _contexts(cuda, cache, rows, n, prefill).float()
    assert bool(torch.isfinite(out).all()) and float(out.abs().max()) <= 1e-30       # 1e30 x 2^-230 is 6e-40


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("n", [500, 30000])
def test_huge_values_of_even_weight(cuda, prefill, n):
    """The mean of values of 1e36: their sum, which the states of a split sequence stand for, is over fp32's largest."""
    v = 1e36 * (1.0 + 0.25 * torch.randn(8, n, 64, generator=torch.Generator().manual_seed(2)))
    cache, ref = _line(cuda, torch.zeros(n), v, room=80)
    rows = _rows(70 if prefill else 4, 241, cuda)
    rows[:, 1536:2048] = (rows[:, 1536:2048].float() * 1e36).to(BF16)
    out = _contexts(cuda, cache, rows, n, prefill)
    table = cache.block_tables()[0].cpu()
    q, k, val = ora.split(rows)
    ora.append(ref, table, n, k, val)
    ora.check_context(out, *ora.attend(ref, table, n, q))


@pytest.mark.parametrize("tokens", [1, 3, 70])
@pytest.mark.parametrize("packed", [False, True])
def test_a_sequence_of_no_token_is_skipped_whatever_its_lengths(cuda, tokens, packed):
    """Slots of a batch that nobody uses: their lengths, rows and tables may be left over."""
    a8, _, lib = _mods()
    lens, chunk = [70, -9, 10 ** 6, 5, 2 ** 31 - 1], [tokens, 0, 0, 1, 0]
    live = (0, 3)
    cache, ref = _build([max(0, min(n, 200)) for n in lens], cuda, seed=251, room=80)
    tables = cache.block_tables()
    tables[1] = -1
    tables[2] = 1 << 30
    b = len(lens)
    rows = _rows(b * tokens, 252, cuda)
    starts = [tokens * i for i in range(b)]
    err, out = _err(cuda), torch.full((b * tokens, 16, 64), -7.0, dtype=BF16, device=cuda)
    args = dict(block_tables=tables, workspace=a8.workspace_kv8(cuda), dev_err=err, mode=lib.B2_STORE_KV,
                chunk_lens=_ints(chunk, cuda), **cache.kv8())
    shape = (rows.to(cuda), out)
    if packed:
        args |= dict(row_start=_ints([0, -50, 10 ** 6, starts[3], 2 ** 31 - 1], cuda), max_tokens=tokens)
    else:
        shape = (rows.to(cuda).view(b, tokens, 2048), out.view(b, tokens, 16, 64))
    if tokens > 4:
        if packed:
            slots = [-1] * (b * tokens)
            for i in live:
                for t in range(chunk[i]):
                    p = lens[i] + t
                    slots[starts[i] + t] = int(tables[i, p // BLOCK]) * BLOCK + p % BLOCK
            args["slots"] = _ints(slots, cuda)
        a8.prefill_kv8(shape[0], _ints(lens, cuda), out=shape[1], **args)
    else:
        a8.decode_step_kv8(shape[0], _ints(lens, cuda), out=shape[1], **args)
    assert err.item() == 0
    seen = torch.zeros(b * tokens, dtype=torch.bool)
    for i in live:
        n, r = chunk[i], starts[i]
        q, k, v = ora.split(rows[r:r + n])
        ora.append(ref, tables[i].cpu(), lens[i], k, v)
        ora.check_context(out[r:r + n], *ora.attend(ref, tables[i].cpu(), lens[i], q), f"sequence {i}")
        seen[r:r + n] = True
    assert bool((out[~seen.to(cuda)] == -7.0).all())
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("gap", [1, 7, 31, 32, 33, 300])
def test_rows_of_a_block_behind_skipped_rows_are_refused(cuda, gap):
    """Skipped rows stand between runs of different blocks; a block whose rows they part is written by its first run
    alone, whichever rows of the call share a CTA."""
    a8, _, lib = _mods()
    lens = [100, 30, 64, 7]
    cache, ref = _build(lens, cuda, seed=261, room=100)
    tables = cache.block_tables()

    def slots_of(b, t0, n):
        return [int(tables[b, p // BLOCK]) * BLOCK + p % BLOCK for p in range(lens[b] + t0, lens[b] + t0 + n)]
    skip = [-1] * gap
    parts = [(0, 0, 5), (0, 5, 3), (1, 0, 34), (1, 34, 20), (2, 0, 2), (3, 0, 1)]
    #        100..104   105..107    30..63     64..: own    another sequence's blocks
    slots, kept, row = [], [], 3
    for b, t0, n in parts:
        slots += skip + slots_of(b, t0, n)
        row = len(slots) - n
        if (b, t0) != (0, 5):                               # goes on in block 1 of sequence 0
            kept.append((b, t0, n, row))
    rows = _rows(len(slots), 262, cuda, sigma=20.0)
    err = _err(cuda)
    q_out = torch.full((len(slots), 16, 64), -7.0, dtype=BF16, device=cuda)
    a8.append_kv8(rows.to(cuda), slots=_ints(slots, cuda), dev_err=err, q_out=q_out, mode=lib.B2_STORE_KV, **cache.kv8())
    assert err.item() == lib.B2_DEV_BAD_SLOT
    for b, t0, n, r in kept:
        _, k, v = ora.split(rows[r:r + n])
        ora.append(ref, tables[b].cpu(), lens[b] + t0, k, v)
    assert ref.same_as(cache.kv8())
    # in one piece nothing is refused
    cache2, ref2 = _build(lens, cuda, seed=261, room=100)
    slots = slots_of(0, 0, 8) + skip + slots_of(1, 0, 54) + slots_of(2, 0, 2) + skip
    rows = _rows(len(slots), 263, cuda)
    err.zero_()
    a8.append_kv8(rows.to(cuda), slots=_ints(slots, cuda), dev_err=err, mode=lib.B2_STORE_KV, **cache2.kv8())
    for b, n, r in ((0, 8, 0), (1, 54, 8 + gap), (2, 2, 62 + gap)):
        _, k, v = ora.split(rows[r:r + n])
        ora.append(ref2, tables[b].cpu(), lens[b], k, v)
    assert err.item() == 0 and ref2.same_as(cache2.kv8())
