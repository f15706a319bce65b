"""The 8-bit paged cache on a B200: codes and scales bit for bit, contexts
within the rounding the kernels make (kv8_oracle.check_context)."""
import itertools

import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg
from oracle import lfm2_attention as orc

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
BLOCK = 64


def _mods():
    return load_pkg("attention_kv8"), load_pkg("paged_cache"), load_pkg("_lib")


def _build(lengths, dev, seed=0, room=8, v_spread=0.0):
    """A PagedKVCache8 full of NaN codes and scales with random histories, and its CPU copy."""
    _, pc, _ = _mods()
    cap = max(lengths) + room
    cache = pc.PagedKVCache8(len(lengths) * pc.blocks_for(cap) + 2, cap, device=dev, shuffle_seed=seed + 1,
                             fill=float("nan"))
    g = torch.Generator().manual_seed(seed)
    for i, n in enumerate(lengths):
        cache.add_sequence(n)
        k = torch.randn(8, n, 64, generator=g)
        v = torch.randn(8, n, 64, generator=g) * torch.exp(v_spread * torch.randn(8, n, 1, generator=g))
        cache.write_dense(0, i, k.to(BF16), v.to(BF16))
    return cache, ora.Cache.of(cache.kv8())


def _rows(n, seed, dev, width=2048, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g) * sigma * torch.exp(0.5 * torch.randn(n, 1, generator=g))
    return x.to(BF16)


def _err(dev):
    return torch.zeros(1, dtype=I32, device=dev)


def _ints(x, dev):
    return torch.tensor(x, dtype=I32, device=dev)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("by_slots", [False, True])
@pytest.mark.parametrize("past,n", [(0, 1), (0, 64), (0, 65), (1, 1), (63, 1), (63, 2), (64, 3), (5, 59), (5, 60),
                                    (17, 200), (130, 7)])
def test_append_codes_and_scales(cuda, past, n, by_slots):
    """Growing and steady scales, block edges; rows behind the last one and other blocks stay as they were."""
    a8, pc, lib = _mods()
    cache, ref = _build([past, past + 3], cuda, seed=past + n, room=260)
    rows = torch.stack([_rows(n, 1, cuda, sigma=s) for s in (0.5, 30.0)])       # the second raises its scales
    err, tables = _err(cuda), cache.block_tables()
    kw = dict(dev_err=err, mode=lib.B2_STORE_KV, **cache.kv8())
    lens = [past, past + 3]
    if by_slots:
        slots = [int(tables[b, (p + t) // BLOCK]) * BLOCK + (p + t) % BLOCK for b, p in enumerate(lens)
                 for t in range(n)]
        a8.append_kv8(rows.reshape(2 * n, -1).to(cuda), slots=_ints(slots, cuda), **kw)
    else:
        a8.append_kv8(rows.to(cuda), past_lens=_ints(lens, cuda), block_tables=tables, **kw)
    for b, p in enumerate(lens):
        _, k, v = ora.split(rows[b])
        ora.append(ref, tables[b].cpu(), p, k, v)
    assert err.item() == 0
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("b,n", [(130, 16), (67, 17), (300, 3)])
def test_append_of_many_short_runs(cuda, b, n):
    a8, pc, lib = _mods()
    lens = [(7 * i) % 70 for i in range(b)]
    cache, ref = _build(lens, cuda, seed=n, room=n)
    rows, err, tables = _rows(b * n, n, cuda).view(b, n, 2048), _err(cuda), cache.block_tables()
    a8.append_kv8(rows.to(cuda), past_lens=_ints(lens, cuda), block_tables=tables, dev_err=err, mode=lib.B2_STORE_KV,
                  **cache.kv8())
    for i, p in enumerate(lens):
        _, k, v = ora.split(rows[i])
        ora.append(ref, tables[i].cpu(), p, k, v)
    assert err.item() == 0
    assert ref.same_as(cache.kv8())


def test_append_skips_negative_slots_and_strange_values(cuda):
    """Negative slots are padding; zeros, tiny, huge, infinite and NaN values have their codes and scales."""
    a8, _, lib = _mods()
    cache, ref = _build([0, 0, 0, 0], cuda, seed=3, room=70)
    tables = cache.block_tables()
    rows = _rows(4 * 6, 2, cuda).view(4, 6, 2048)
    rows[0, :] = 0
    rows[1, :, :] *= 1e-38
    rows[2, 1] = float("inf")
    rows[2, 2, 1024:] = -3.3e38
    rows[3, 0] = float("nan")
    rows[3, 4, 1100] = float("-inf")
    slots, flat = [], []
    for b in range(4):
        slots += [int(tables[b, 0]) * BLOCK + t for t in range(6)] + [-1]
        flat += [rows[b], torch.full((1, 2048), 7.0, dtype=BF16)]
    err = _err(cuda)
    a8.append_kv8(torch.cat(flat).to(cuda), slots=_ints(slots, cuda), dev_err=err, mode=lib.B2_STORE_KV,
                  **cache.kv8())
    for b in range(4):
        _, k, v = ora.split(rows[b])
        ora.append(ref, tables[b].cpu(), 0, k, v)
    assert err.item() == 0
    got = ora.Cache.of(cache.kv8())
    for x, y in ((got.k, ref.k), (got.v, ref.v)):
        assert torch.equal(x.float().nan_to_num(999.0), y.float().nan_to_num(999.0))
    assert torch.equal(got.ks.nan_to_num(-1.0), ref.ks.nan_to_num(-1.0))
    assert torch.equal(got.vs.nan_to_num(-1.0), ref.vs.nan_to_num(-1.0))


def test_append_one_by_one_raises_scales_like_a_chunk(cuda):
    """Powers of two: a block filled token by token ends with the scales of one append, and the codes too
    wherever the larger scale does not make them subnormal."""
    a8, _, lib = _mods()
    one, _ = _build([0], cuda, seed=4, room=70)
    two, _ = _build([0], cuda, seed=4, room=70)
    rows = _rows(70, 5, cuda).to(cuda)
    err = _err(cuda)
    a8.append_kv8(rows[None], past_lens=_ints([0], cuda), block_tables=one.block_tables(), dev_err=err,
                  mode=lib.B2_STORE_KV, **one.kv8())
    for t in range(70):
        a8.append_kv8(rows[None, t:t + 1].contiguous(), past_lens=_ints([t], cuda), block_tables=two.block_tables(),
                      dev_err=err, mode=lib.B2_STORE_KV, **two.kv8())
    used = one.block_tables()[0].long()
    assert torch.equal(one.k_scale[0, used], two.k_scale[0, used])
    assert torch.equal(one.v_scale[0, used], two.v_scale[0, used])
    x, y = one.read_dense(0, 0, 70)[0].float(), two.read_dense(0, 0, 70)[0].float()
    step = one.k_scale[0, used].max() * 2.0 ** -9          # the spacing of subnormal codes
    assert bool(((x - y).abs() <= step).all()) and float((x != y).float().mean()) < 0.02


def test_append_norm_rope_matches_oracle(cuda):
    a8, _, _ = _mods()
    lengths = [0, 1, 63, 64, 200]
    cache, ref = _build(lengths, cuda, seed=6)
    w = orc.attention_weights(0)
    rows = _rows(5 * 3, 7, cuda).view(5, 3, 2048)
    cos, sin = load_pkg("rope").rope_table(256, device=cuda)
    q_out = torch.zeros(15, 16, 64, dtype=BF16, device=cuda)
    err, tables = _err(cuda), cache.block_tables()
    a8.append_kv8(rows.to(cuda), past_lens=_ints(lengths, cuda), block_tables=tables, dev_err=err, q_out=q_out,
                  gamma_q=w["q_gamma"].to(cuda), gamma_k=w["k_gamma"].to(cuda), cos=cos, sin=sin, **cache.kv8())
    assert err.item() == 0
    for b, p in enumerate(lengths):
        q, k, v = ora.split(rows[b])
        q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin([p, p + 1, p + 2]))
        assert torch.equal(q_out.view(5, 3, 16, 64)[b].cpu(), q)
        ora.append(ref, tables[b].cpu(), p, k, v)
    assert ref.same_as(cache.kv8())


# ------------------------------------------------------------------ decode step

def _step(cache, rows, lens, dev, chunk=None, mode=None, out=None, work=None, **kw):
    a8, _, lib = _mods()
    b, t = rows.shape[:2]
    err = _err(dev)
    out = torch.full((b, t, 16, 64), -7.0, dtype=BF16, device=dev) if out is None else out
    a8.decode_step_kv8(rows.to(dev), _ints(lens, dev), block_tables=cache.block_tables(), out=out,
                       workspace=a8.workspace_kv8(dev) if work is None else work, dev_err=err,
                       chunk_lens=None if chunk is None else _ints(chunk, dev),
                       mode=lib.B2_STORE_KV if mode is None else mode, **cache.kv8(), **kw)
    assert err.item() == 0
    return out


def _check_step(cache, ref, rows, lens, chunk, out, what=""):
    tables = cache.block_tables().cpu()
    for b, p in enumerate(lens):
        n = rows.shape[1] if chunk is None else chunk[b]
        if n:
            q, k, v = ora.split(rows[b, :n])
            ora.append(ref, tables[b], p, k, v)
            ora.check_context(out[b, :n], *ora.attend(ref, tables[b], p, q), f"{what} sequence {b}")
        assert bool((out[b, n:] == -7.0).all()), f"rows past sequence {b}'s chunk were written"
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("tokens", [1, 2, 3, 4])
@pytest.mark.parametrize("lens", [[0], [37], [0, 1, 62, 63, 64, 65, 127, 128, 300], [1000, 5, 2047], [4095]])
def test_step(cuda, lens, tokens):
    cache, ref = _build(lens, cuda, seed=len(lens) + tokens, v_spread=0.5)
    rows = _rows(len(lens) * tokens, 11, cuda).view(len(lens), tokens, 2048)
    _check_step(cache, ref, rows, lens, None, _step(cache, rows, lens, cuda))


def test_step_ragged_and_waiting_sequences(cuda):
    lens = [70, 0, 63, 5, 200, 64, 128]
    chunk = [4, 0, 3, 1, 0, 2, 4]
    cache, ref = _build(lens, cuda, seed=21)
    rows = _rows(28, 12, cuda).view(7, 4, 2048)
    _check_step(cache, ref, rows, lens, chunk, _step(cache, rows, lens, cuda, chunk))
    # nobody has a token: nothing is written
    out = _step(cache, rows, lens, cuda, [0] * 7)
    assert bool((out == -7.0).all()) and ref.same_as(cache.kv8())


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("width", [2048, 2304])
def test_step_norm_rope_and_wide_rows(cuda, tokens, width):
    lens = [0, 63, 129]
    cache, ref = _build(lens, cuda, seed=31)
    w = orc.attention_weights(1)
    rows = _rows(3 * tokens, 13, cuda, width).view(3, tokens, width)
    cos, sin = load_pkg("rope").rope_table(256, device=cuda)
    out = _step(cache, rows, lens, cuda, mode=7, gamma_q=w["q_gamma"].to(cuda), gamma_k=w["k_gamma"].to(cuda), cos=cos,
                sin=sin)
    tables = cache.block_tables().cpu()
    for b, p in enumerate(lens):
        q, k, v = ora.split(rows[b])
        q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin(list(range(p, p + tokens))))
        ora.append(ref, tables[b], p, k, v)
        ora.check_context(out[b], *ora.attend(ref, tables[b], p, q))
    assert ref.same_as(cache.kv8())


def test_step_without_store_reads_the_tokens_in_the_cache(cuda):
    lens = [64, 10]
    cache, ref = _build([n + 2 for n in lens], cuda, seed=41)
    rows = _rows(4, 14, cuda).view(2, 2, 2048)
    out = _step(cache, rows, lens, cuda, mode=0)
    for b, p in enumerate(lens):
        ora.check_context(out[b], *ora.attend(ref, cache.block_tables()[b].cpu(), p, ora.split(rows[b])[0]))
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("tokens", [1, 4])
def test_step_merges_across_ctas(cuda, tokens):
    """Long sequences beside short ones: segments of many CTAs, of some warps and of parts of one."""
    lens = [30000, 3, 700, 64, 12001, 0, 129]
    cache, ref = _build(lens, cuda, seed=51)
    rows = _rows(7 * tokens, 15, cuda).view(7, tokens, 2048)
    work = _mods()[0].workspace_kv8(cuda)
    out = _step(cache, rows, lens, cuda, work=work)
    _check_step(cache, ref, rows, lens, None, out)
    assert bool((work[:4096] == 0).all())          # the counters are ready for the next call
    again = _step(cache, rows, lens, cuda, work=work)
    assert torch.equal(out, again)                 # appending the same tokens again changes nothing


def test_step_more_sequences_than_one_launch_takes(cuda):
    lens = [(7 * i) % 90 for i in range(1500)]
    cache, ref = _build(lens, cuda, seed=61)
    rows = _rows(1500, 16, cuda).view(1500, 1, 2048)
    chunk = [0 if i % 11 == 3 else 1 for i in range(1500)]
    out = _step(cache, rows, lens, cuda, chunk)
    tables = cache.block_tables().cpu()
    for b in itertools.chain(range(0, 40), range(1010, 1040), range(1480, 1500)):
        if chunk[b]:
            q, k, v = ora.split(rows[b])
            ora.append(ref, tables[b], lens[b], k, v)
            ora.check_context(out[b], *ora.attend(ref, tables[b], lens[b], q), f"sequence {b}")
        else:
            assert bool((out[b] == -7.0).all())


def _scaled_history(cuda, factors_k, factors_v, seed, rows_sigma=1.0):
    """One sequence whose blocks have the given magnitudes."""
    _, pc, _ = _mods()
    nb = len(factors_k)
    cache = pc.PagedKVCache8(nb + 2, (nb + 1) * BLOCK, device=cuda, fill=float("nan"))
    cache.add_sequence(nb * BLOCK)
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(8, nb, BLOCK, 64, generator=g) * torch.tensor(factors_k).view(1, nb, 1, 1)
    v = torch.randn(8, nb, BLOCK, 64, generator=g) * torch.tensor(factors_v).view(1, nb, 1, 1)
    cache.write_dense(0, 0, k.reshape(8, -1, 64).to(BF16), v.reshape(8, -1, 64).to(BF16))
    return cache, ora.Cache.of(cache.kv8())


@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("order", [1, -1])
def test_step_scales_far_apart(cuda, order, tokens):
    """Blocks of very different V magnitudes whose weights are of the opposite order, blocks of zeros and
    growing scores: neither reference may flush what counts."""
    fv = [1e-6, 0.0, 1.0, 3e5, 1e-3, 2.0, 1e8, 1e-8, 1.0][::order]
    fk = [8.0, 1.0, 4.0, 0.05, 6.0, 2.0, 0.01, 9.0, 1.0][::order]
    cache, ref = _scaled_history(cuda, fk, fv, 71)
    rows = _rows(tokens, 17, cuda, sigma=0.7).view(1, tokens, 2048)
    _check_step(cache, ref, rows, [9 * BLOCK], None, _step(cache, rows, [9 * BLOCK], cuda))


def test_step_large_scores_and_queries(cuda):
    """Scores of hundreds (one key takes all) and queries at the ends of bf16's range."""
    cache, ref = _build([400, 130, 70], cuda, seed=81)
    rows = _rows(3, 18, cuda).view(3, 1, 2048)
    rows[0, 0, :1024] *= 60
    rows[1, 0, :1024] = (rows[1, 0, :1024].float() * 1e-30).to(BF16)
    rows[2, 0, :1024] = 0
    _check_step(cache, ref, rows, [400, 130, 70], None, _step(cache, rows, [400, 130, 70], cuda))


def test_step_faults_are_flagged_and_not_performed(cuda):
    a8, _, lib = _mods()
    lens = [100, 200, 30]
    cache, ref = _build(lens, cuda, seed=91)
    rows = _rows(3, 19, cuda).view(3, 1, 2048).to(cuda)
    out = torch.zeros(3, 1, 16, 64, dtype=BF16, device=cuda)
    work = a8.workspace_kv8(cuda)

    def run(tables, past, chunk=None):
        err = _err(cuda)
        a8.decode_step_kv8(rows, _ints(past, cuda), block_tables=tables, out=out, workspace=work, dev_err=err,
                           chunk_lens=None if chunk is None else _ints(chunk, cuda), mode=lib.B2_STORE_KV,
                           **cache.kv8())
        return err.item()
    for bad in (-1, cache.num_blocks, 1 << 30):
        tables = cache.block_tables()
        tables[0, 1], tables[1, 0], tables[2, 0] = bad, bad, bad
        assert run(tables, lens) == lib.B2_DEV_BAD_BLOCK
    # the appends with a good block were made, the others were not
    _, k, v = ora.split(rows[1].cpu())
    ora.append(ref, cache.block_tables()[1].cpu(), 200, k, v)
    assert ref.same_as(cache.kv8())
    width = cache.block_tables().shape[1]
    assert run(cache.block_tables(), [width * BLOCK, -1, 30]) == lib.B2_DEV_BAD_LENGTH
    assert run(cache.block_tables(), lens, [2, -1, 1]) == lib.B2_DEV_BAD_LENGTH
    assert run(cache.block_tables(), lens) == 0


# ------------------------------------------------------------------ prompt chunks

def _prefill(cache, rows, lens, dev, chunk=None, mode=None, **kw):
    a8, _, lib = _mods()
    err = _err(dev)
    out = a8.prefill_kv8(rows.to(dev), _ints(lens, dev), block_tables=cache.block_tables(),
                         workspace=a8.workspace_kv8(dev), dev_err=err,
                         chunk_lens=None if chunk is None else _ints(chunk, dev),
                         mode=lib.B2_STORE_KV if mode is None else mode, **cache.kv8(), **kw)
    assert err.item() == 0
    return out


def _check_rows(cache, ref, rows, out, lens, starts, counts):
    tables = cache.block_tables().cpu()
    seen = torch.zeros(rows.shape[0], dtype=torch.bool)
    for b, (p, r, n) in enumerate(zip(lens, starts, counts)):
        q, k, v = ora.split(rows[r:r + n])
        if n:
            ora.append(ref, tables[b], p, k, v)
            ora.check_context(out[r:r + n], *ora.attend(ref, tables[b], p, q), f"sequence {b}")
        seen[r:r + n] = True
    assert bool((out[~seen.to(out.device)] == 0).all()), "rows of no token were written"
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("lens,tokens", [([0], 1), ([0], 21), ([0], 64), ([0, 3], 65), ([63, 64, 1], 63),
                                         ([130, 0, 500], 200), ([2000], 5), ([9000], 33), ([300] * 20, 130)])
def test_prefill_padded(cuda, lens, tokens):
    """One tile, several tiles, split keys (few long sequences) and none (many)."""
    cache, ref = _build(lens, cuda, seed=tokens, room=tokens + 3, v_spread=0.5)
    rows = _rows(len(lens) * tokens, 22, cuda)
    out = _prefill(cache, rows.view(len(lens), tokens, 2048), lens, cuda)
    _check_rows(cache, ref, rows, out.view(-1, 16, 64), lens, [b * tokens for b in range(len(lens))],
                [tokens] * len(lens))


def test_prefill_padded_ragged(cuda):
    lens, chunk = [10, 64, 0, 700], [70, 1, 0, 33]
    cache, ref = _build(lens, cuda, seed=101, room=80)
    rows = _rows(4 * 70, 23, cuda)
    out = _prefill(cache, rows.view(4, 70, 2048), lens, cuda, chunk)
    _check_rows(cache, ref, rows, out.view(-1, 16, 64), lens, [0, 70, 140, 210], chunk)


@pytest.mark.parametrize("norm_rope", [False, True])
def test_prefill_packed(cuda, norm_rope):
    """Prompts behind one another through a slot map, with rows of no token between and behind them."""
    a8, pc, lib = _mods()
    bt = load_pkg("block_tables")
    lens, chunk, starts = [5, 0, 130, 64, 63], [100, 1, 65, 0, 190], [0, 100, 104, 169, 169]
    cache, ref = _build(lens, cuda, seed=111, room=200)
    rows = _rows(365, 24, cuda)
    slots, positions = _ints([9] * 365, cuda), _ints([9] * 365, cuda)
    err = _err(cuda)
    bt.slot_map(cache.block_tables(), _ints(lens, cuda), _ints(chunk, cuda), num_blocks=cache.num_blocks, slots=slots,
                positions=positions, row_start=_ints(starts, cuda), dev_err=err)
    kw = dict(row_start=_ints(starts, cuda), max_tokens=190, slots=slots, positions=positions)
    if not norm_rope:
        out = _prefill(cache, rows, lens, cuda, chunk, **kw)
        _check_rows(cache, ref, rows, out, lens, starts, chunk)
        return
    w = orc.attention_weights(2)
    cos, sin = load_pkg("rope").rope_table(512, device=cuda)
    out = _prefill(cache, rows, lens, cuda, chunk, mode=7, gamma_q=w["q_gamma"].to(cuda),
                   gamma_k=w["k_gamma"].to(cuda), cos=cos, sin=sin, **kw)
    turned = rows.clone()
    for p, r, n in zip(lens, starts, chunk):
        if n:
            q, k, v = ora.split(rows[r:r + n])
            q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin(list(range(p, p + n))))
            turned[r:r + n] = torch.cat([q.reshape(n, -1), k.reshape(n, -1), v.reshape(n, -1)], 1)
    _check_rows(cache, ref, turned, out, lens, starts, chunk)


@pytest.mark.parametrize("top", [1, 2, 4])
@pytest.mark.parametrize("norm_rope", [False, True])
@pytest.mark.parametrize("binding", [True, False])
def test_step_packed(cuda, top, norm_rope, binding, monkeypatch):
    """Packed rows with gaps and empty chunks; a sequence behind the last row is refused, the others are not."""
    a8, _, lib = _mods()
    if not binding:
        monkeypatch.setattr(a8, "_b2torch", None)
    lens, chunk, starts = [5, 0, 130, 64, 63], [top, 1, top, 0, 1], [1, 1 + top, 4 + top, 4 + 2 * top, 4 + 2 * top]
    n = 6 + 2 * top
    cache, ref = _build(lens, cuda, seed=113, room=20)
    rows = _rows(n, 31, cuda)
    kw = dict(row_start=_ints(starts, cuda), max_tokens=top)
    turned = rows.clone()
    if norm_rope:
        w = orc.attention_weights(5)
        cos, sin = load_pkg("rope").rope_table(256, device=cuda)
        kw |= dict(mode=7, gamma_q=w["q_gamma"].to(cuda), gamma_k=w["k_gamma"].to(cuda), cos=cos, sin=sin)
        for p, r, m in zip(lens, starts, chunk):
            if m:
                q, k, v = ora.split(rows[r:r + m])
                q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin(list(range(p, p + m))))
                turned[r:r + m] = torch.cat([q.reshape(m, -1), k.reshape(m, -1), v.reshape(m, -1)], 1)
    out = torch.zeros(n, 16, 64, dtype=BF16, device=cuda)
    kept = [t.clone() for t in cache.kv8().values()]
    for last, flagged in ((n, True), (starts[4], False)):
        # the refused call first: it leaves its own sequence and only that one out
        for t, was in zip(cache.kv8().values(), kept):
            t.copy_(was)
        out.zero_()
        kw["row_start"] = _ints(starts[:4] + [last], cuda)
        err = _err(cuda)
        a8.decode_step_kv8(rows.to(cuda), _ints(lens, cuda), block_tables=cache.block_tables(), out=out,
                           workspace=a8.workspace_kv8(cuda), dev_err=err, chunk_lens=_ints(chunk, cuda),
                           **{"mode": lib.B2_STORE_KV, **kw}, **cache.kv8())
        assert err.item() == (lib.B2_DEV_BAD_LENGTH if flagged else 0)
        if flagged:
            assert not bool(out[starts[4]:].any())
    _check_rows(cache, ref, turned, out, lens, starts, chunk)
    call = dict(block_tables=cache.block_tables(), out=out, workspace=a8.workspace_kv8(cuda), dev_err=_err(cuda),
                **{"mode": lib.B2_STORE_KV, **kw}, **cache.kv8())
    for bad in (dict(row_start=None), dict(max_tokens=None), dict(max_tokens=0), dict(max_tokens=5),
                dict(row_start=_ints(starts[:4], cuda)), dict(row_start=_ints(starts, "cpu")), dict(out=out[:-1])):
        with pytest.raises(ValueError):
            a8.decode_step_kv8(rows.to(cuda), _ints(lens, cuda), **{**call, **bad})
    with pytest.raises(ValueError):
        a8.decode_step_kv8(rows.to(cuda).view(1, n, 2048), _ints(lens, cuda), **call)
    if norm_rope:
        runner = a8.PagedDecodeAttentionKV8(cache, kw["gamma_q"], kw["gamma_k"], n, 256)
        for t, was in zip(cache.kv8().values(), kept):
            t.copy_(was)
        got = runner.step(0, rows.to(cuda), _ints(lens, cuda), cache.block_tables(), chunk_lens=_ints(chunk, cuda),
                          row_start=kw["row_start"], max_tokens=top)
        runner.check()
        assert torch.equal(got, out)
        with pytest.raises(ValueError, match="row_start"):
            runner.step(0, rows.to(cuda), _ints(lens, cuda), cache.block_tables(), max_tokens=top)
        with pytest.raises(ValueError, match="rows"):
            runner.step(0, torch.zeros(n + 1, 2048, dtype=BF16, device=cuda), _ints(lens, cuda), cache.block_tables(),
                        row_start=kw["row_start"], max_tokens=top)


def test_step_packed_of_many_sequences(cuda):
    """More sequences than one launch takes, some without a new token: as the padded call."""
    a8, _, lib = _mods()
    n = 2100
    lens = [(11 * i) % 90 for i in range(n)]
    chunk = [(i % 5 > 0) + (i % 7 == 0) for i in range(n)]
    starts = [sum(chunk[:b]) for b in range(n)]
    cache, _ = _build(lens, cuda, seed=8, room=3)
    kept = [t.clone() for t in cache.kv8().values()]
    rows = _rows(sum(chunk), 8, cuda)
    padded = torch.zeros(n, 2, 2048, dtype=BF16)
    for b in range(n):
        padded[b, :chunk[b]] = rows[starts[b]:starts[b] + chunk[b]]
    want = _step(cache, padded, lens, cuda, chunk)
    after = [t.clone().view(torch.uint8) for t in cache.kv8().values()]
    for t, was in zip(cache.kv8().values(), kept):
        t.copy_(was)
    out = torch.full((sum(chunk), 16, 64), -7.0, dtype=BF16, device=cuda)
    err = _err(cuda)
    a8.decode_step_kv8(rows.to(cuda), _ints(lens, cuda), block_tables=cache.block_tables(), out=out, dev_err=err,
                       workspace=a8.workspace_kv8(cuda), chunk_lens=_ints(chunk, cuda), mode=lib.B2_STORE_KV,
                       row_start=_ints(starts, cuda), max_tokens=2, **cache.kv8())
    assert err.item() == 0
    assert all(torch.equal(x.view(torch.uint8), y) for x, y in zip(cache.kv8().values(), after))
    there = torch.arange(2)[None] < torch.tensor(chunk)[:, None]
    assert torch.equal(out, want[there.to(cuda)])


@pytest.mark.parametrize("n", [9, 33, 64, 65, 128, 129])
def test_prefill_packed_many_ragged(cuda, n):
    """More query tiles than start at once: sorted by their blocks, or (more than 128 sequences) as they come; a
    sequence whose chunk passes max_tokens is refused, the others are not."""
    a8, _, lib = _mods()
    g = torch.Generator().manual_seed(n)
    top = 700 if n < 30 else 140
    lens = torch.randint(0, 300, (n,), generator=g).tolist()
    chunk = torch.randint(0, top + 1, (n,), generator=g).tolist()
    chunk[0], chunk[1], chunk[n // 2], lens[2] = 0, top, 64, 64
    starts = [sum(chunk[:b]) for b in range(n)]
    cache, ref = _build(lens, cuda, seed=n, room=top + 1)
    rows = _rows(sum(chunk), n, cuda)
    slots = torch.full((sum(chunk),), -1, dtype=I32)
    tables = cache.block_tables().cpu()
    for b in range(n):
        for t in range(chunk[b]):
            p = lens[b] + t
            slots[starts[b] + t] = int(tables[b, p // 64]) * 64 + p % 64
    kw = dict(row_start=_ints(starts, cuda), max_tokens=top, slots=slots.to(cuda))
    out = _prefill(cache, rows, lens, cuda, chunk, **kw)
    want = out.clone()
    _check_rows(cache, ref, rows, out, lens, starts, chunk)
    err, out = _err(cuda), torch.zeros_like(out)
    bad = [top + 1 if b == 1 else c for b, c in enumerate(chunk)]
    a8.prefill_kv8(rows.to(cuda), _ints(lens, cuda), block_tables=cache.block_tables(), dev_err=err, out=out,
                   workspace=a8.workspace_kv8(cuda), chunk_lens=_ints(bad, cuda), mode=0, **cache.kv8(), **kw)
    assert err.item() == lib.B2_DEV_BAD_LENGTH
    want[starts[1]:starts[1] + top] = 0
    assert torch.equal(out, want)


def test_prefill_packed_with_a_loose_bound(cuda):
    """max_tokens may be any bound of the chunks."""
    a8, _, _ = _mods()
    cache, ref = _build([70, 3], cuda, seed=115, room=80)
    rows = _rows(60, 30, cuda)
    tables = cache.block_tables()
    slots = [int(tables[0, (70 + t) // BLOCK]) * BLOCK + (70 + t) % BLOCK for t in range(40)]
    slots += [int(tables[1, 0]) * BLOCK + 3 + t for t in range(20)]
    out = _prefill(cache, rows, [70, 3], cuda, [40, 20], row_start=_ints([0, 40], cuda), max_tokens=2 ** 31 - 1,
                   slots=_ints(slots, cuda))
    _check_rows(cache, ref, rows, out, [70, 3], [0, 40], [40, 20])


@pytest.mark.parametrize("order", [1, -1])
def test_prefill_scales_far_apart(cuda, order):
    fv = [1e-6, 0.0, 1.0, 3e5, 1e-3, 2.0, 1e8, 1e-8, 1.0][::order]
    fk = [8.0, 1.0, 4.0, 0.05, 6.0, 2.0, 0.01, 9.0, 1.0][::order]
    cache, ref = _scaled_history(cuda, fk, fv, 121)
    rows = _rows(60, 25, cuda, sigma=0.7)
    out = _prefill(cache, rows.view(1, 60, 2048), [9 * BLOCK], cuda)
    _check_rows(cache, ref, rows, out.view(-1, 16, 64), [9 * BLOCK], [0], [60])


def test_prefill_in_chunks_then_steps(cuda):
    """A prompt in three chunks, then decode steps and drafted tokens, over the same cache."""
    lens, cache, ref = [0, 40], *_build([0, 40], cuda, seed=131, room=400)
    tables = cache.block_tables().cpu()
    work = _mods()[0].workspace_kv8(cuda)
    for i, t in enumerate([100, 64, 7, 1, 4, 1, 2]):
        rows = _rows(2 * t, 26 + i, cuda).view(2, t, 2048)
        out = _prefill(cache, rows, lens, cuda) if i < 3 else _step(cache, rows, lens, cuda, work=work)
        for b in range(2):
            q, k, v = ora.split(rows[b])
            ora.append(ref, tables[b], lens[b], k, v)
            ora.check_context(out[b], *ora.attend(ref, tables[b], lens[b], q), f"call {i}")
            lens[b] += t
    assert ref.same_as(cache.kv8())


def test_prefill_faults_are_flagged(cuda):
    a8, _, lib = _mods()
    cache, _ = _build([100, 30], cuda, seed=141, room=200)
    rows = _rows(2 * 70, 27, cuda).view(2, 70, 2048).to(cuda)

    def run(tables, past, chunk=None, qkv=rows, **kw):
        err = _err(cuda)
        a8.prefill_kv8(qkv, _ints(past, cuda), block_tables=tables, workspace=a8.workspace_kv8(cuda), dev_err=err,
                       chunk_lens=None if chunk is None else _ints(chunk, cuda), mode=lib.B2_STORE_KV, **cache.kv8(),
                       **kw)
        return err.item()
    tables = cache.block_tables()
    tables[0, 0] = cache.num_blocks
    assert run(tables, [100, 30]) == lib.B2_DEV_BAD_BLOCK
    width = tables.shape[1]
    assert run(cache.block_tables(), [100, width * BLOCK - 69]) == lib.B2_DEV_BAD_LENGTH
    assert run(cache.block_tables(), [100, -5]) == lib.B2_DEV_BAD_LENGTH
    assert run(cache.block_tables(), [100, 30], [71, 3]) == lib.B2_DEV_BAD_LENGTH
    # packed rows behind the last one, a slot behind the pool
    flat, slots = rows.view(140, 2048), _ints([-1] * 140, cuda)
    kw = dict(row_start=_ints([0, 80], cuda), max_tokens=70, positions=slots, qkv=flat)
    assert run(cache.block_tables(), [100, 30], [70, 70], slots=slots, **kw) == lib.B2_DEV_BAD_LENGTH
    slots[3] = cache.num_blocks * BLOCK
    assert run(cache.block_tables(), [100, 30], [70, 60], slots=slots, **kw) == lib.B2_DEV_BAD_BLOCK
    assert run(cache.block_tables(), [100, 30]) == 0


# ------------------------------------------------------------------ streams, graphs, the runner

def test_step_on_another_stream_and_two_at_once(cuda):
    """Two runners' steps on two streams, each with its own workspace."""
    a8, _, lib = _mods()
    jobs = []
    for s in range(2):
        lens = [3000 + 700 * s, 50, 64]
        cache, ref = _build(lens, cuda, seed=151 + s)
        rows = _rows(3, 28 + s, cuda).view(3, 1, 2048)
        jobs.append((lens, cache, ref, rows, rows.to(cuda), cache.block_tables(), a8.workspace_kv8(cuda), _err(cuda),
                     torch.full((3, 1, 16, 64), -7.0, dtype=BF16, device=cuda), _ints(lens, cuda)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in jobs]
    for _ in range(5):
        for st, (lens, cache, ref, rows, dev_rows, tables, work, err, out, past) in zip(streams, jobs):
            a8.decode_step_kv8(dev_rows, past, block_tables=tables, out=out, workspace=work, dev_err=err,
                               mode=lib.B2_STORE_KV, stream=st, **cache.kv8())
    torch.cuda.synchronize()
    for lens, cache, ref, rows, _, _, _, err, out, _ in jobs:
        assert err.item() == 0
        _check_step(cache, ref, rows, lens, None, out)


def test_runner_step_in_a_graph(cuda):
    """PagedDecodeAttentionKV8.step captured once and replayed while the lengths move across a block's edge."""
    a8, _, _ = _mods()
    lens = [60, 0, 126]
    cache, ref = _build(lens, cuda, seed=161, room=40)
    w = orc.attention_weights(3)
    runner = a8.PagedDecodeAttentionKV8(cache, w["q_gamma"], w["k_gamma"], 3, 256)
    tables = cache.block_tables()
    past, qkv = _ints(lens, cuda), torch.zeros(3, 2048, dtype=BF16, device=cuda)
    start = ora.Cache.of(cache.kv8())
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        runner.step(0, qkv, past, tables)              # warm-up: appends zeros, undone below
    torch.cuda.synchronize()
    for name, t in (("k_pool", start.k), ("v_pool", start.v), ("k_scale", start.ks), ("v_scale", start.vs)):
        dst = cache.kv8()[name]
        (dst.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else dst).copy_(
            t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = runner.step(0, qkv, past, tables)
        past.add_(1)
    for i in range(8):
        rows = _rows(3, 40 + i, cuda)
        qkv.copy_(rows)
        graph.replay()
        runner.check()
        for b in range(3):
            q, k, v = ora.split(rows[b:b + 1])
            q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin([lens[b]]))
            ora.append(ref, tables[b].cpu(), lens[b], k, v)
            ora.check_context(out[b:b + 1], *ora.attend(ref, tables[b].cpu(), lens[b], q), f"replay {i}")
            lens[b] += 1
    assert ref.same_as(cache.kv8())


def test_serving_loop_allocates_in_a_graph(cuda):
    """The set together: device block tables give blocks on demand, packed prompts go through the slot map,
    decode steps allocate, append and attend in one captured graph; a finished request's blocks are reused."""
    a8, pc, lib = _mods()
    bt = load_pkg("block_tables")
    b, blocks = 4, 9
    cache = pc.PagedKVCache8(blocks, 256, device=cuda, fill=float("nan"))
    ref = ora.Cache.of(cache.kv8())
    dev = bt.DeviceBlockTables(b, blocks, 256, cuda)
    work, err = a8.workspace_kv8(cuda), _err(cuda)
    # prompts: request 3 waits
    new = [70, 3, 64, 0]
    rows = _rows(150, 50, cuda)
    plan = dev.plan(_ints(new, cuda), rows=150)
    out = a8.prefill_kv8(rows.to(cuda), dev.lens, block_tables=dev.tables, row_start=plan.row_start, max_tokens=128,
                         chunk_lens=plan.granted, slots=plan.slots, positions=plan.positions, workspace=work,
                         dev_err=err, mode=lib.B2_STORE_KV, **cache.kv8())
    dev.advance(plan)
    lens = [0] * b
    assert plan.granted.tolist() == new
    tables = dev.tables.cpu()
    r = 0
    for i, n in enumerate(new):
        if n:
            q, k, v = ora.split(rows[r:r + n])
            ora.append(ref, tables[i], 0, k, v)
            ora.check_context(out[r:r + n], *ora.attend(ref, tables[i], 0, q), f"prompt {i}")
        r += n
        lens[i] = n
    # decode: one token each per replay
    qkv = torch.zeros(b, 1, 2048, dtype=BF16, device=cuda)
    ctx = torch.full((b, 1, 16, 64), -7.0, dtype=BF16, device=cuda)
    want = _ints([1, 1, 1, 0], cuda)
    step_plan = dev.plan(_ints([0] * b, cuda), tokens_per_seq=1)

    def step():
        dev.plan(want, tokens_per_seq=1, out=step_plan)
        a8.decode_step_kv8(qkv, dev.lens, block_tables=dev.tables, out=ctx, workspace=work, dev_err=err,
                           chunk_lens=step_plan.granted, mode=lib.B2_STORE_KV, **cache.kv8())
        dev.advance(step_plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(70):
        if i == 40:       # request 1 ends, request 3 starts in its place
            dev.release(torch.tensor([False, True, False, False], device=cuda))
            want.copy_(_ints([1, 0, 1, 1], cuda))
            lens[1] = 0
        x = _rows(b, 60 + i, cuda).view(b, 1, 2048)
        qkv.copy_(x)
        graph.replay()
        tables = dev.tables.cpu()
        for j in range(b):
            if not int(want[j]):
                continue
            assert int(step_plan.granted[j]) == 1
            q, k, v = ora.split(x[j])
            ora.append(ref, tables[j], lens[j], k, v)
            ora.check_context(ctx[j], *ora.attend(ref, tables[j], lens[j], q), f"step {i} request {j}")
            lens[j] += 1
    assert err.item() == 0
    dev.check()
    assert dev.lens.tolist() == lens
    held = [int(t) for t in dev.tables.flatten() if t >= 0]
    free = dev.free_list[:int(dev.free_count)].tolist()
    assert sorted(held + free) == list(range(blocks))
    assert ref.same_as(cache.kv8())


@pytest.mark.parametrize("binding", [True, False])
def test_native_binding_and_python_checks_agree(cuda, binding, monkeypatch):
    """The same calls and the same refusals with the native binding and without it."""
    a8, _, lib = _mods()
    assert a8._b2torch is not None, "the native binding is not built"
    if not binding:
        monkeypatch.setattr(a8, "_b2torch", None)
    bt = load_pkg("block_tables")
    lens = [5, 64]
    cache, ref = _build(lens, cuda, seed=171, room=80)
    w = orc.attention_weights(4)
    cos, sin = load_pkg("rope").rope_table(256, device=cuda)
    qk = dict(gamma_q=w["q_gamma"].to(cuda), gamma_k=w["k_gamma"].to(cuda), cos=cos, sin=sin)
    for n, call in ((1, _step), (70, _prefill)):
        rows = _rows(2 * n, 70 + n, cuda).view(2, n, 2048)
        out = call(cache, rows, lens, cuda, mode=7, **qk)
        for b, p in enumerate(lens):
            q, k, v = ora.split(rows[b])
            q, k = orc.norm_rope_qk(q, k, w["q_gamma"], w["k_gamma"], *orc.rope_cos_sin(list(range(p, p + n))))
            ora.append(ref, cache.block_tables()[b].cpu(), p, k, v)
            ora.check_context(out[b], *ora.attend(ref, cache.block_tables()[b].cpu(), p, q))
        lens = [p + n for p in lens]
    assert ref.same_as(cache.kv8())
    good = dict(block_tables=cache.block_tables(), workspace=a8.workspace_kv8(cuda), dev_err=_err(cuda), **cache.kv8())
    rows, past = _rows(2, 1, cuda).view(2, 1, 2048).to(cuda), _ints(lens, cuda)
    out = torch.zeros(2, 1, 16, 64, dtype=BF16, device=cuda)
    for name, bad in (("block_tables", good["block_tables"].cpu()), ("block_tables", good["block_tables"].long()),
                      ("k_scale", cache.k_scale[0].T), ("v_pool", cache.k[0][:-1]), ("workspace", out),
                      ("dev_err", _ints([0, 0], cuda)), ("chunk_lens", past.cpu()), ("gamma_q", None)):
        with pytest.raises(ValueError):
            a8.decode_step_kv8(rows, past, out=out, mode=7, **{**qk, **good, name: bad})
        if name != "chunk_lens":
            with pytest.raises(ValueError):
                a8.prefill_kv8(rows, past, out=out, mode=7, **{**qk, **good, name: bad})
    with pytest.raises(lib.B2Error, match="workspace"):
        a8.decode_step_kv8(rows, past, out=out, **{**qk, **good, "workspace": good["workspace"][:64]})
    with pytest.raises(lib.B2Error, match="scale"):
        a8.decode_step_kv8(rows, past, out=out, scale=-1.0, **qk, **good)
    # a parameter is a tensor too; whole numbers as scale
    a8.decode_step_kv8(torch.nn.Parameter(rows, requires_grad=False), past, out=out, scale=1, **qk, **good)
    dev = bt.DeviceBlockTables(2, 4, 128, cuda)
    plan = dev.plan(_ints([64, 65], cuda), rows=129)
    assert plan.granted.tolist() == [64, 65] and dev.held.tolist() == [1, 2]
    with pytest.raises(ValueError):
        dev.plan(_ints([1, 1, 1], cuda), rows=3)


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("given", [True, False])
def test_prefill_on_another_stream(cuda, binding, given, monkeypatch):
    """The call's own buffers belong to the stream it runs on: work that the current stream is given meanwhile
    does not get them."""
    a8, _, lib = _mods()
    if not binding:
        monkeypatch.setattr(a8, "_b2torch", None)
    cache, _ = _build([70, 3], cuda, seed=19, room=80)
    w = orc.attention_weights(6)
    cos, sin = load_pkg("rope").rope_table(256, device=cuda)
    rows, past = _rows(140, 19, cuda).view(2, 70, 2048).to(cuda), _ints([70, 3], cuda)
    args = dict(block_tables=cache.block_tables(), workspace=a8.workspace_kv8(cuda), dev_err=_err(cuda),
                gamma_q=w["q_gamma"].to(cuda), gamma_k=w["k_gamma"].to(cuda), cos=cos, sin=sin, mode=7, **cache.kv8())
    want = a8.prefill_kv8(rows, past, **args)
    out = torch.zeros_like(want) if given else None
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    got = a8.prefill_kv8(rows, past, out=out, stream=side, **args)
    junk = [torch.full((140, 16, 64), float("nan"), dtype=BF16, device=cuda) for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and args["dev_err"].item() == 0 and bool(junk[0].isnan().all())


def test_refuses_host_tensors(cuda):
    """Tensors that are all on the host never reach the library."""
    a8, pc, lib = _mods()
    cache = pc.PagedKVCache8(2, 64, device="cpu")
    args = dict(block_tables=torch.zeros(1, 1, dtype=I32), out=torch.zeros(1, 1, 16, 64, dtype=BF16),
                workspace=torch.zeros(64, dtype=torch.uint8), dev_err=torch.zeros(1, dtype=I32), mode=lib.B2_STORE_KV,
                **cache.kv8())
    with pytest.raises(ValueError, match="CUDA device"):
        a8.decode_step_kv8(torch.zeros(1, 1, 2048, dtype=BF16), torch.zeros(1, dtype=I32), **args)
