"""Host checks of the 8-bit cache and the device block tables: refusals before any launch, the cache's set-up
path against the plain restatement, the ABI's argument errors."""
import ctypes

import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg

BF16, I32 = torch.bfloat16, torch.int32


def _step_args(b=2, t=1, blocks=6, width=3):
    a8 = load_pkg("attention_kv8")
    pc = load_pkg("paged_cache")
    cache = pc.PagedKVCache8(blocks, width * 64, device="cpu", fill=0.0)
    return a8, {"qkv": torch.zeros(b, t, 2048, dtype=BF16), "past_lens": torch.zeros(b, dtype=I32),
                "block_tables": torch.zeros(b, width, dtype=I32), "out": torch.zeros(b, t, 16, 64, dtype=BF16),
                "workspace": torch.zeros(1024, dtype=torch.uint8), "dev_err": torch.zeros(1, dtype=I32),
                "mode": load_pkg("_lib").B2_STORE_KV, **cache.kv8()}


@pytest.mark.parametrize("name,value,text", [
    ("qkv", torch.zeros(2, 1, 2040, dtype=BF16), "qkv"),
    ("qkv", torch.zeros(2, 1, 2048), "qkv"),
    ("qkv", torch.zeros(2, 5, 2048, dtype=BF16), "tokens"),
    ("qkv", torch.zeros(2, 1, 4096, dtype=BF16)[:, :, ::2], "contiguous"),
    ("past_lens", torch.zeros(2, dtype=torch.int64), "past_lens"),
    ("past_lens", torch.zeros(3, dtype=I32), "past_lens"),
    ("chunk_lens", torch.zeros(1, dtype=I32), "chunk_lens"),
    ("block_tables", torch.zeros(3, 3, dtype=I32), "past_lens"),
    ("block_tables", torch.zeros(6, dtype=I32), "block_tables"),
    ("out", torch.zeros(2, 16, 64, dtype=BF16), "out"),
    ("workspace", torch.zeros(1024), "workspace"),
    ("k_pool", torch.zeros(6, 8, 64, 64, dtype=BF16), "k_pool"),
    ("v_pool", torch.zeros(5, 8, 64, 64, dtype=torch.float8_e4m3fn), "v_pool"),
    ("k_scale", torch.zeros(6, 8, dtype=BF16), "k_scale"),
    ("v_scale", torch.zeros(6, 4), "v_scale"),
    ("mode", 7, "gamma_q"),
])
def test_step_refusals(name, value, text):
    a8, args = _step_args()
    args[name] = value
    with pytest.raises(ValueError, match=text):
        a8.decode_step_kv8(args.pop("qkv"), args.pop("past_lens"), **args)


def test_prefill_and_append_refusals():
    a8, args = _step_args(t=9)
    del args["out"]
    qkv, past = args.pop("qkv"), args.pop("past_lens")
    with pytest.raises(ValueError, match="row_start"):
        a8.prefill_kv8(qkv, past, row_start=past, **args)
    with pytest.raises(ValueError, match="packed"):
        a8.prefill_kv8(qkv.view(18, 2048), past, **args)
    with pytest.raises(ValueError, match="out"):
        a8.prefill_kv8(qkv, past, out=torch.zeros(18, 16, 64, dtype=BF16), **args)
    with pytest.raises(ValueError, match="padded"):
        a8.prefill_kv8(qkv[:1].contiguous(), past, **args)
    kw = {k: args[k] for k in ("k_pool", "v_pool", "k_scale", "v_scale", "dev_err", "mode")}
    with pytest.raises(ValueError, match="without slots"):
        a8.append_kv8(qkv.view(18, 2048), past_lens=past, block_tables=args["block_tables"], **kw)
    with pytest.raises(ValueError, match="slots"):
        a8.append_kv8(qkv.view(18, 2048), slots=torch.zeros(17, dtype=I32), **kw)
    with pytest.raises(ValueError, match="rows"):
        a8.append_kv8(qkv[:1].contiguous(), past_lens=past, block_tables=args["block_tables"], **kw)
    pc = load_pkg("paged_cache")
    with pytest.raises(ValueError, match="PagedKVCache8"):
        a8.PagedDecodeAttentionKV8(pc.PagedKVCache(2, 64, device="cpu"), torch.ones(64), torch.ones(64), 1, 8)


def test_bf16_wrappers_refuse_the_8_bit_cache():
    attn = load_pkg("attention")
    _, args = _step_args()
    with pytest.raises(ValueError, match="k_pool"):
        attn.decode_step(args["qkv"][:, 0].contiguous(), args["past_lens"], k_pool=args["k_pool"],
                         v_pool=args["v_pool"], block_tables=args["block_tables"], blocks_per_split=1, out=None,
                         part_ml=None, part_o=None, counters=None, dev_err=args["dev_err"])


def test_table_refusals():
    bt = load_pkg("block_tables")

    def ints(*shape):
        return torch.zeros(*shape, dtype=I32)
    good = dict(granted=ints(2), row_start=ints(2), slots=ints(4), positions=ints(4), dev_err=ints(1))
    state = (ints(2, 3), ints(2), ints(8), ints(1), ints(2), ints(2))
    for i, bad in ((0, ints(6)), (1, ints(3)), (2, ints(8).float()), (3, ints(2)), (4, ints(1)), (5, ints(2).long())):
        args = list(state)
        args[i] = bad
        with pytest.raises(ValueError):
            bt.extend_tables(*args, **good)
    for k, bad in (("granted", ints(3)), ("row_start", ints(1)), ("positions", ints(5)), ("slots", ints(4).long()),
                   ("dev_err", ints(2)), ("held_out", ints(1)), ("free_count_out", ints(2))):
        with pytest.raises(ValueError):
            bt.extend_tables(*state, **{**good, k: bad})
    with pytest.raises(ValueError):
        bt.release_tables(*state[:4], ints(2), dev_err=ints(1))
    with pytest.raises(ValueError):
        bt.slot_map(ints(2, 3), ints(2), ints(3), num_blocks=8, slots=ints(4), positions=ints(4), dev_err=ints(1))
    with pytest.raises(ValueError):
        bt.DeviceBlockTables(0, 4, 64, "cpu")
    with pytest.raises(ValueError, match="rows"):
        bt.DeviceBlockTables(2, 4, 64, "cpu").plan(ints(2))


def test_abi_argument_errors_without_gpu():
    lib = load_pkg("_lib")
    c = lib.load()
    f = ctypes.c_float
    raw = ctypes.create_string_buffer(256)
    buf = (ctypes.addressof(raw) + 63) & ~63
    nbytes = c.b2_kv8_workspace_bytes()
    assert nbytes > 0

    def refused(rc, text):
        assert rc == lib.B2_ERR_ARG, rc
        assert text in lib.last_error(), lib.last_error()

    def step(qkv=buf, stride=2048, tokens=1, width=4, k=buf, ks=buf, blocks=8, batch=1, scale=0.125, mode=4, out=buf,
             ws=buf, size=nbytes, gamma=None, rope=None, rows=64, start=None):
        return c.b2_kv8_decode_step(qkv, stride, rows, start, tokens, None, gamma, gamma, f(1e-5), rope, rope, 0, buf, buf, width, k,
                                    buf, ks, buf, blocks, batch, f(scale), mode, out, ws, size, buf, None)
    refused(step(tokens=5), "tokens")
    refused(step(tokens=0), "tokens")
    refused(step(batch=-1), "batch")
    refused(step(rows=-1, start=buf), "rows")
    refused(step(batch=17, tokens=4, rows=67), "row_start")
    refused(step(stride=2044), "row_stride")
    refused(step(qkv=buf + 8), "qkv")
    refused(step(width=1 << 25), "max_blocks_per_seq")
    refused(step(k=buf + 4), "aligned")
    refused(step(ks=buf + 4), "aligned")
    refused(step(k=None), "null")
    refused(step(blocks=0), "num_blocks")
    refused(step(blocks=1 << 22), "num_blocks")
    refused(step(scale=0.0), "scale")
    refused(step(scale=float("nan")), "scale")
    refused(step(mode=0x104), "mode")
    refused(step(mode=5), "gamma")
    refused(step(mode=6), "cos/sin")
    refused(step(out=None), "out")
    refused(step(size=nbytes - 1), "workspace")
    refused(step(ws=buf + 8), "workspace")
    assert step(batch=0) == lib.B2_OK

    def append(rows=6, slots=None, positions=None, tokens=3, tables=buf, q_out=None, mode=4, rope=None):
        return c.b2_kv8_append(buf, 2048, rows, slots, positions, buf, None, tokens, tables, 4, None, None, f(1e-5),
                               rope, rope, 8, buf, buf, buf, buf, 8, q_out, mode, buf, None)
    refused(append(rows=7), "multiple")
    refused(append(tokens=0), "multiple")
    refused(append(tables=None), "block_tables")
    refused(append(mode=0), "nothing to write")
    refused(append(slots=buf, mode=6, rope=buf), "positions")
    assert append(rows=0) == lib.B2_OK

    def prefill(stride=1024, rows=6, start=None, tokens=3, batch=2, out=buf, size=nbytes):
        return c.b2_kv8_prefill_attn(buf, stride, rows, start, buf, None, tokens, buf, 4, buf, buf, buf, buf, 8, batch,
                                     f(0.125), out, buf, size, buf, None)
    refused(prefill(stride=1020), "q_stride")
    refused(prefill(rows=5), "row_start")
    refused(prefill(batch=65536, start=buf), "65535")
    refused(prefill(out=buf + 2), "aligned")
    refused(prefill(size=0), "workspace")
    assert prefill(batch=0) == lib.B2_OK and prefill(tokens=0) == lib.B2_OK

    def extend(batch=2, rows=6, tokens=3, width=4, blocks=8, slots=buf):
        return c.b2_tables_extend(buf, width, buf, buf, blocks, buf, buf, buf, batch, buf, buf, buf, buf, slots, buf,
                                  rows, tokens, buf, None)
    refused(extend(rows=5), "tokens_per_seq")
    refused(extend(batch=-1), "batch")
    refused(extend(width=0), "max_blocks_per_seq")
    refused(extend(blocks=1 << 22), "num_blocks")
    refused(extend(slots=None), "null")
    refused(c.b2_slot_map(buf, 4, 8, buf, buf, None, 2, buf, buf, 6, 0, buf, None), "row_start")
    refused(c.b2_tables_release(buf, 4, None, buf, 8, buf, buf, 2, buf, None), "null")
    assert c.b2_tables_release(buf, 4, buf, buf, 8, buf, buf, 0, buf, None) == lib.B2_OK


@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 200])
def test_write_dense_is_one_append(length):
    pc = load_pkg("paged_cache")
    cache = pc.PagedKVCache8(8, 256, device="cpu", fill=float("nan"), shuffle_seed=5)
    cache.add_sequence(length, capacity=256)
    ref = ora.Cache.of(cache.kv8())
    g = torch.Generator().manual_seed(length)
    k, v = (torch.randn(8, length, 64, generator=g) * s for s in (1.0, 40.0))
    k, v = k.to(BF16), v.to(BF16)
    cache.write_dense(0, 0, k, v)
    if length:
        ora.append(ref, cache.block_tables()[0], 0, k.transpose(0, 1), v.transpose(0, 1))
    got_k, got_v = cache.read_dense(0, 0, length)
    want_k, want_v = ora.values(ref, cache.block_tables()[0], length)
    assert torch.equal(got_k.double(), want_k) and torch.equal(got_v.double(), want_v)
    assert torch.equal(cache.k_scale[0].nan_to_num(-1), ref.ks.nan_to_num(-1))
    # a code is off by at most half a step, 2^-4 of the value, or half the spacing of subnormal codes
    off = (got_k.double() - k.double()).abs()
    tiny = cache.k_scale[0].nan_to_num(0).max().double() * 2.0 ** -10
    assert bool((off <= torch.maximum(k.double().abs() * 2.0 ** -4, tiny)).all())


def test_scale_is_the_smallest_power_of_two():
    pc = load_pkg("paged_cache")
    x = torch.tensor([0.0, 1e-40, 2.0 ** -100 * 448, 1.0, 447.9, 448.0, 448.1, 896.0, 3.3e38])
    s = pc.kv8_scale(x)
    assert s.tolist() == [ora.scale_of(float(v)) for v in x]
    x, s = x.double(), s.double()                       # 448 * s may pass the largest fp32
    assert bool((x <= 448 * s).all())
    big = s > 2.0 ** -100
    assert bool((x[big] > 448 * s[big] / 2).all())


def test_cache_needs_half_the_bytes():
    pc = load_pkg("paged_cache")
    full, half = pc.PagedKVCache(16, 256, device="cpu"), pc.PagedKVCache8(16, 256, device="cpu")
    size = {id(c): sum(t.numel() * t.element_size() for t in (c.k, c.v)) for c in (full, half)}
    assert size[id(full)] == 2 * size[id(half)]
