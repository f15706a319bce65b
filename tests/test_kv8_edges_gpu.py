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
