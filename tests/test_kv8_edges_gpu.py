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
