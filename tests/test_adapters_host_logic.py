"""Host side of the adapters' plan and bank, and the refusals that need no GPU."""
import random

import pytest
import torch

from more4d_amd import _lib, ops


def tables(p):
    base, t, a = p.table.data_ptr(), p.table.tolist(), p.args

    def at(ptr, n):
        o = (ptr - base) // 4
        assert (ptr - base) % 64 == 0 and o + n <= len(t)
        return t[o:o + n]
    return at, a


@pytest.mark.parametrize("seed", range(12))
def test_plan_tables_cover_every_row_once(seed):
    rng = random.Random(seed)
    n = rng.choice([1, 2, 7, 300])
    lengths = [rng.choice([0, 1, 1, 5, 63, 64, 65, 300]) for _ in range(n)]
    ids = [rng.randint(-1, 6) for _ in range(n)]
    p = ops.AdapterPlan(lengths, ids, "cpu")
    at, a = tables(p)
    rows = [i for k, i in zip(lengths, ids) for _ in range(k)]
    assert p.rows == a.rows == len(rows) and at(a.row_adapter, len(rows)) == rows
    slots, pieces = at(a.slot_row, 64 * p.n_pieces), at(a.piece_adapter, p.n_pieces)
    assert sorted(s for s in slots if s >= 0) == [r for r, i in enumerate(rows) if i >= 0]
    for q, g in enumerate(pieces):
        own = slots[64 * q:64 * q + 64]
        assert own[0] >= 0 and all(rows[s] == g for s in own if s >= 0)
        assert all(s >= 0 for s in own) or q == p.n_pieces - 1 or pieces[q + 1] != g       # only an adapter's last piece is padded
    assert p.n_adapters == max(rows, default=-1) + 1
    for level in range(4):
        n = a.n_chunks[level]
        off = at(a.chunk_off[level], p.n_adapters + 1)
        ch = at(a.chunks[level], 3 * n)
        assert off[0] == 0 and off[-1] == n
        covered = []
        for g in range(p.n_adapters):
            for c in range(off[g], off[g + 1]):
                assert ch[3 * c + 2] == g and 0 < ch[3 * c + 1] - ch[3 * c] <= 64
                covered += range(ch[3 * c], ch[3 * c + 1])
                assert all(pieces[q] == g for q in range(ch[3 * c], ch[3 * c + 1]))
        assert covered == list(range(p.n_pieces))
    order = at(a.row_order, len(rows)) if a.row_order else list(range(len(rows)))
    assert sorted(order) == list(range(len(rows))) and (not a.row_order or [rows[r] for r in order] == sorted(rows))
    in_order = [rows[r] for r in order]
    for k, T in enumerate((64, 128, 256, 256)):
        of_tiles = rows if k == 3 else in_order
        nt = -(-p.rows // T)
        off = at(a.tiles_off[k], nt + 1)
        lst = at(a.tiles[k], off[-1])
        for i in range(nt):
            lo = max(0, min(i * T, p.rows - T)) if k == 3 else i * T
            assert lst[off[i]:off[i + 1]] == sorted({g for g in of_tiles[lo:i * T + T] if g >= 0})
            if k == 3:
                here = set(rows[lo:i * T + T])
                assert at(a.tile_one, nt)[i] == (here.pop() if len(here) == 1 else -1)
    assert a.n_listed == at(a.tiles_off[0], -(-p.rows // 64) + 1)[-1] and a.n_wide == at(a.tiles_off[3], -(-p.rows // 256) + 1)[-1]


def test_interleaved_requests_are_tiled_in_order_of_their_adapters():
    p = ops.AdapterPlan([1] * 256, [i % 8 for i in range(256)], "cpu")
    at, a = tables(p)
    assert at(a.row_order, 256) == sorted(range(256), key=lambda r: r % 8) and a.n_listed == 8 and a.n_wide == 8
    assert ops.AdapterPlan([32] * 8, list(range(8)), "cpu").args.row_order is None
    assert ops.AdapterPlan([1] * 64, [i % 8 for i in range(64)], "cpu").args.row_order is None       # one tile either way


def test_plan_of_nothing():
    for lengths, ids in (([], []), ([0], [3]), ([5], [-1])):
        p = ops.AdapterPlan(lengths, ids, "cpu")
        assert p.n_pieces == p.n_adapters == 0 and list(p.args.n_chunks) == [0] * 4 and p.rows == sum(lengths)


def test_plan_refusals():
    for lengths, ids in (([1, 2], [0]), ([-1], [0]), ([1], [-2]), ([1 << 30, 1 << 30], [-1, -1])):
        with pytest.raises(ValueError):
            ops.AdapterPlan(lengths, ids, "cpu")


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    a, b = torch.randn(1, 4, 64), torch.randn(1, 32, 4)
    with pytest.raises(_lib.More4DHipError):
        ops.AdapterBank(a, b, [1.0])
    with pytest.raises(_lib.More4DHipError):
        ops.act_quant8(x)
    with pytest.raises(ValueError):
        ops.act_quant8(torch.empty(4, 0))
    with pytest.raises(TypeError):
        ops.act_quant8(x.half())


@pytest.mark.parametrize("dtype,K,fits,too_wide", [(torch.float32, 64, (64,), (68, 72)), (torch.float32, 61, (61, 64), (60, 68)), (torch.bfloat16, 64, (64,), (72,)),
                                                   (torch.bfloat16, 60, (60, 64), (56, 68, 72))])
def test_rows_padded_by_more_than_one_chunk_are_refused(dtype, K, fits, too_wide):
    """The bank is laid out in chunks of 64 channels: a row that reaches into one more would read the next adapter's, or behind the bank."""
    bank = ops.AdapterBank.__new__(ops.AdapterBank)
    bank.buf, bank.K, bank.G = torch.empty(0, dtype=dtype), K, 1
    plan = ops.AdapterPlan([3], [0], "cpu")
    for k in fits:
        assert ops._check_adapters("test", torch.zeros(3, k, dtype=dtype), bank, plan) == (3, k)
    for k in too_wide:
        with pytest.raises(ValueError):
            ops._check_adapters("test", torch.zeros(3, k, dtype=dtype), bank, plan)


def test_adapter_numbers_have_a_limit():
    """(the tables hold an entry per adapter number: a stray one would ask for all the memory there is)"""
    assert ops.AdapterPlan([1], [65534], "cpu").n_adapters == 65535
    for i in (65535, 1 << 31, 1 << 40):
        with pytest.raises(ValueError):
            ops.AdapterPlan([0], [i], "cpu")
    a, b = torch.empty(1).expand(65536, 1, 1), torch.empty(1).expand(65536, 1, 1)
    with pytest.raises(ValueError):
        ops.AdapterBank(a, b, [1.0] * 65536)


def test_slots_of_another_type_than_the_bank_are_refused():
    """bfloat16 slots hold two parts per value, float32 slots one: read as the other type they would end before the kernel does."""
    bank = ops.AdapterBank.__new__(ops.AdapterBank)
    plan = ops.AdapterPlan([3], [0], "cpu")
    bank.G, bank.rank, bank.R = 1, 4, 16
    for own, other in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        bank.buf = torch.empty(0, dtype=own)
        with pytest.raises(TypeError):
            ops.adapter_grad(torch.zeros(ops._slots_shape(bank, plan), dtype=other), torch.zeros(3, 64, dtype=other), plan, bank)


def test_a_buffer_that_is_not_whole_is_refused():
    """Act8's kernels address its buffer as n bytes one behind the other."""
    n = 2 * 33
    assert ops.Act8((2, 32), torch.float32, buf=torch.empty(n, dtype=torch.uint8)).rows == 2
    for buf in (torch.empty(n + 1, dtype=torch.uint8), torch.empty(1, dtype=torch.uint8).expand(n), torch.empty(2 * n, dtype=torch.uint8)[::2],
                torch.empty(n, dtype=torch.int8)):
        with pytest.raises(ValueError):
            ops.Act8((2, 32), torch.float32, buf=buf)


def test_side_libraries_are_built_with_the_flags_of_the_library(tmp_path):
    """tools/side_lib.sh compiles one source to stand in for the library's: with another flag list (packed float32 instructions on) it would not."""
    import os
    import subprocess
    from more4d_amd.build import FLAGS
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    stub, log = tmp_path / "hipcc", tmp_path / "log"
    stub.write_text(f'#!/bin/bash\nprintf "%s\\n" "$*" >> {log}\n')
    stub.chmod(0o755)
    subprocess.run(["bash", os.path.join(root, "tools", "side_lib.sh"), "x", "act8.hip", "-DY=1"], check=True, env={**os.environ, "HIPCC": str(stub)},
                   capture_output=True)
    line = log.read_text().splitlines()[0].split()
    assert set(FLAGS) <= set(line) and "-DY=1" in line and "-DM4D_ABLATIONS" in line
