"""Block tables and slot maps built on the GPU against the same rules on Python lists."""
import random

import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _ints(x, dev):
    return torch.tensor(x, dtype=I32, device=dev)


def _state(b, width, blocks, rng, past):
    """held blocks for `past`, the rest on the free list in a random order."""
    ids = list(range(blocks))
    rng.shuffle(ids)
    held = [-(-max(p, 0) // 64) for p in past]
    tables = []
    for h in held:
        tables.append([ids.pop() for _ in range(h)] + [-1] * (width - h))
    return tables, held, ids


def _run(dev, tables, held, free, blocks, past, new, rows, tps, in_place=False, count=None):
    bt = load_pkg("block_tables")
    b = len(tables)
    t = _ints(tables, dev).view(b, -1)
    free_list = _ints(free + [-9] * (blocks - len(free)), dev)
    c = _ints([len(free) if count is None else count], dev)
    h, err = _ints(held, dev), _ints([0], dev)
    out = {k: torch.full((n,), -5, dtype=I32, device=dev) for k, n in
           (("granted", b), ("row_start", b), ("slots", rows), ("positions", rows))}
    ho, co = (None, None) if in_place else (torch.full_like(h, -5), torch.full_like(c, -5))
    bt.extend_tables(t, h, free_list, c, _ints(past, dev), _ints(new, dev), held_out=ho, free_count_out=co,
                     tokens_per_seq=tps, dev_err=err, **out)
    if not in_place:
        assert h.tolist() == held and c.item() == (len(free) if count is None else count)
    got = {k: v.tolist() for k, v in out.items()}
    got |= {"tables": t.tolist(), "held": (h if in_place else ho).tolist(), "count": (c if in_place else co).item(),
            "bad": bool(err.item() & load_pkg("_lib").B2_DEV_BAD_LENGTH)}
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("b,top,tight", [(1, 1, False), (1, 5000, False), (7, 70, False), (7, 300, True), (64, 1, False),
                                         (1023, 9, True), (1025, 130, False), (3000, 66, True)])
def test_extend(cuda, b, top, tight, packed, in_place):
    rng = random.Random(b * 1000 + top + packed)
    past = [rng.randint(0, 200) for _ in range(b)]
    new = [rng.randint(0 if b > 1 else top, top) for _ in range(b)]
    width = (200 + top + 63) // 64
    need = sum(-(-(p + n) // 64) for p, n in zip(past, new))
    have = sum(-(-p // 64) for p in past)
    blocks = have + ((need - have) // 2 if tight else need - have) + 1
    tables, held, free = _state(b, width, blocks, rng, past)
    rows = sum(new) + 3 if packed else b * top
    want = ora.extend(tables, held, free, len(free), past, new, rows, 0 if packed else top)
    got = _run(cuda, tables, held, free, blocks, past, new, rows, 0 if packed else top, in_place)
    assert got == want


@pytest.mark.parametrize("b,top,packed", [(293, 1801, False), (911, 1301, True), (3, 200001, True)])
def test_extend_many_rows(cuda, b, top, packed):
    """Above half a million rows: several per thread, requests that end inside a thread's rows."""
    test_extend(cuda, b, top, False, packed, False)


def test_extend_refuses_what_cannot_be(cuda):
    """Negative lengths, a full row, rows behind the last one, more tokens than a padded row has: refused, the
    others served."""
    rng = random.Random(5)
    past = [10, -1, 64, 300, 20, 100, 0]
    new = [5, 3, -2, 21, 4, 60, 9]
    tables, held, free = _state(7, 5, 40, rng, past)
    for rows, tps in ((200, 0), (60, 0), (7 * 30, 30)):
        want = ora.extend(tables, held, free, len(free), past, new, rows, tps)
        got = _run(cuda, tables, held, free, 40, past, new, rows, tps)
        assert want["bad"] and 0 in want["granted"]
        live = [i for i, p in enumerate(past) if p >= 0]
        for k in ("tables", "held", "count", "granted", "row_start", "slots", "bad"):
            assert got[k] == want[k], k
        assert live


def test_extend_nothing_to_do(cuda):
    tables, held, free = _state(3, 2, 8, random.Random(1), [64, 0, 5])
    got = _run(cuda, tables, held, free, 8, [64, 0, 5], [0, 0, 0], 4, 0)
    assert got["slots"] == [-1] * 4 and got["tables"] == tables and got["count"] == len(free)
    bt = load_pkg("block_tables")                       # no request at all
    err, slots = _ints([0], cuda), _ints([3, 3], cuda)
    none = torch.empty(0, dtype=I32, device=cuda)
    count = _ints([4], cuda)
    bt.extend_tables(torch.empty(0, 2, dtype=I32, device=cuda), none, _ints([0, 1, 2, 3], cuda), count, none, none,
                     granted=none, row_start=none, slots=slots, positions=slots.clone(), dev_err=err)
    assert slots.tolist() == [-1, -1] and count.item() == 4 and err.item() == 0


def test_extend_flags_a_bad_free_list(cuda):
    lib = load_pkg("_lib")
    bt = load_pkg("block_tables")
    for ids, count, flag in (([7, 99, 3], 3, lib.B2_DEV_BAD_BLOCK), ([7, -4, 3], 3, lib.B2_DEV_BAD_BLOCK),
                             # a count over the list's size is taken as the size: id 3 of 3 blocks comes first
                             ([1, 2, 3], 5, lib.B2_DEV_BAD_LENGTH | lib.B2_DEV_BAD_BLOCK),
                             ([1, 2, 3], -1, lib.B2_DEV_BAD_LENGTH)):
        err = _ints([0], cuda)
        t = torch.full((1, 4), -1, dtype=I32, device=cuda)
        z = [torch.zeros(1, dtype=I32, device=cuda) for _ in range(3)]
        slots = torch.zeros(128, dtype=I32, device=cuda)
        bt.extend_tables(t, z[0], _ints(ids, cuda), _ints([count], cuda), _ints([0], cuda), _ints([128], cuda),
                         granted=z[1], row_start=z[2], slots=slots, positions=slots.clone(), dev_err=err)
        assert err.item() == flag
        assert bool((t < 3).all())


@pytest.mark.parametrize("b", [1, 5, 700, 2500])
def test_slot_map(cuda, b):
    bt = load_pkg("block_tables")
    rng = random.Random(b)
    past = [rng.randint(0, 300) for _ in range(b)]
    new = [rng.randint(0, 80) for _ in range(b)]
    tables, held, _ = _state(b, 6, 6 * b, rng, [p + n for p, n in zip(past, new)])
    at, starts = 0, []
    for n in new:
        at += rng.randint(0, 2)                         # rows of no token between the requests
        starts.append(at)
        at += n
    rows = at + 4
    want_s, want_p = [-1] * rows, [0] * rows
    for i in range(b):
        for t in range(new[i]):
            pos = past[i] + t
            want_s[starts[i] + t] = tables[i][pos // 64] * 64 + pos % 64
            want_p[starts[i] + t] = pos
    slots, positions, err = _ints([5] * rows, cuda), _ints([5] * rows, cuda), _ints([0], cuda)
    bt.slot_map(_ints(tables, cuda), _ints(past, cuda), _ints(new, cuda), num_blocks=6 * b, slots=slots,
                positions=positions, row_start=_ints(starts, cuda), dev_err=err)
    assert slots.tolist() == want_s and positions.tolist() == want_p and err.item() == 0
    slots, positions = _ints([5] * (80 * b), cuda), _ints([5] * (80 * b), cuda)
    bt.slot_map(_ints(tables, cuda), _ints(past, cuda), _ints(new, cuda), num_blocks=6 * b, slots=slots,
                positions=positions, tokens_per_seq=80, dev_err=err)
    for i in range(b):
        r = starts[i]
        assert slots[80 * i:80 * i + new[i]].tolist() == want_s[r:r + new[i]]
        assert slots[80 * i + new[i]:80 * (i + 1)].tolist() == [-1] * (80 - new[i])
    # a block that is not there, a length that does not fit
    lib = load_pkg("_lib")
    t = _ints(tables, cuda)
    t[b - 1, :] = -1
    new[b - 1] = max(new[b - 1], 1)
    bt.slot_map(t, _ints(past, cuda), _ints(new, cuda), num_blocks=6 * b, slots=slots, positions=positions,
                tokens_per_seq=80, dev_err=err)
    assert err.item() == lib.B2_DEV_BAD_BLOCK
    err.zero_()
    past[0], new[0] = 6 * 64, 1
    bt.slot_map(_ints(tables, cuda), _ints(past, cuda), _ints(new, cuda), num_blocks=6 * b, slots=slots,
                positions=positions, tokens_per_seq=80, dev_err=err)
    assert err.item() & lib.B2_DEV_BAD_LENGTH


@pytest.mark.parametrize("b", [1, 6, 1500])
def test_release_and_reuse(cuda, b):
    bt = load_pkg("block_tables")
    rng = random.Random(b + 9)
    past = [rng.randint(0, 300) for _ in range(b)]
    tables, held, free = _state(b, 5, 5 * b + 2, rng, past)
    done = [rng.random() < 0.5 for _ in range(b)]
    done[0] = True
    blocks = 5 * b + 2
    t, h, err = _ints(tables, cuda), _ints(held, cuda), _ints([0], cuda)
    free_list, count = _ints(free + [-9] * (blocks - len(free)), cuda), _ints([len(free)], cuda)
    bt.release_tables(t, h, free_list, count, torch.tensor(done, device=cuda), dev_err=err)
    back = [x for i in range(b) if done[i] for x in tables[i][:held[i]]]
    assert err.item() == 0
    assert free_list[:len(free) + len(back)].tolist() == free + back and count.item() == len(free) + len(back)
    assert t.tolist() == [[-1] * 5 if done[i] else tables[i] for i in range(b)]
    assert h.tolist() == [0 if done[i] else held[i] for i in range(b)]
    # more ids than the list holds: nothing is released
    h2, t2 = _ints(held, cuda), _ints(tables, cuda)
    full = _ints([blocks], cuda)
    bt.release_tables(t2, h2, free_list, full, torch.ones(b, dtype=torch.bool, device=cuda), dev_err=err)
    if sum(held):
        assert err.item() == load_pkg("_lib").B2_DEV_BAD_LENGTH
    assert h2.tolist() == held and t2.tolist() == tables and full.item() == blocks
