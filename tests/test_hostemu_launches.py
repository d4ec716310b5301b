"""The vocabulary table's launches (CPU, no GPU): the C ABI compiled for x86 over
the HIP emulation lists what it would launch, at sizes that no CPU run has memory
for."""

import struct
from collections import namedtuple

import pytest

from tests.test_hostemu import _exec
from tests.test_hostemu_table import run_table  # noqa: F401

QUANTISE, LOOKUP, GRADIENT, HEAD, DEQUANTISE = 1, 2, 3, 4, 5
F32, BF16, F16, MX4 = 0, 1, 2, 3
ELAUNCH = 3

Launch = namedtuple("Launch", "taken grid threads kernel")


@pytest.fixture
def launches(run_table, tmp_path, monkeypatch):  # noqa: F811
    """The return code and launches of an entry point at given sizes."""
    def call(entry, dtype, out_dtype, n, vocab, hidden, accumulate=0, cus=256):
        inp, out, listed = tmp_path / "in.bin", tmp_path / "out.bin", tmp_path / "launches"
        listed.write_text("")
        inp.write_bytes(struct.pack("<16i", 5, entry, dtype, out_dtype, n, vocab, hidden, accumulate, *[0] * 8))
        monkeypatch.setenv("LPS_EMU_LAUNCHES", str(listed))
        monkeypatch.setenv("LPS_EMU_CUS", str(cus))
        (rc,) = struct.unpack("<i", _exec(run_table, inp, out))
        parts = [x.split(" ", 5) for x in listed.read_text().splitlines()]
        return rc, [Launch(t == "1", (int(x), int(y), int(z)), int(b), f) for t, x, y, z, b, f in parts]
    return call


def fits(rc, made):
    return rc == 0 and len(made) > 0 and all(m.taken for m in made)


@pytest.mark.parametrize("vocab,hidden", [(4096 * 1024 + 1, 1), (1 << 23, 24), ((1 << 31) - 1, 1), (4096 * 1024, 1), (7, 40)])
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
def test_empty_batch_into_a_new_gradient(launches, vocab, hidden, out_dtype):
    """No position: the zeros alone, whatever the vocabulary; nothing when accumulating."""
    rc, made = launches(GRADIENT, BF16, out_dtype, 0, vocab, hidden)
    assert fits(rc, made) and len(made) == 1
    assert launches(GRADIENT, BF16, out_dtype, 0, vocab, hidden, 1) == (0, [])


@pytest.mark.parametrize("n,vocab,hidden,failing", [(3000, 1000, 64, 0), (3000, 1000, 64, 1), (3000, 1000, 64, 2),
                                                    (5, 100000, 1024, 0), (5, 1000, 64, 0)])
def test_nothing_follows_a_failed_launch(launches, monkeypatch, n, vocab, hidden, failing):
    """What a kernel would read is then not there: ids and counts of whatever the memory held."""
    monkeypatch.setenv("LPS_EMU_FAIL", str(failing))
    rc, made = launches(GRADIENT, BF16, F32, n, vocab, hidden)
    assert rc == ELAUNCH and [m.taken for m in made] == [True] * failing + [False]


MANY = 1 << 28    # rows of 16 threads each: 2^32 threads


@pytest.mark.parametrize("rows,hidden,parts", [(MANY - 16, 1, 1), (MANY - 15, 1, 2), (MANY + 5, 1, 2), ((1 << 31) - 1, 1, 9),
                                               ((1 << 24) - 1, 2049, 1), (1 << 24, 2049, 2), (1 << 24, 4096, 2)])
@pytest.mark.parametrize("entry,dtype,out_dtype", [(QUANTISE, BF16, 0), (DEQUANTISE, F16, 0), (LOOKUP, BF16, BF16),
                                                   (LOOKUP, MX4, F16)])
def test_rows_past_a_grid(launches, entry, dtype, out_dtype, rows, hidden, parts):
    """More rows than fewer than 2^32 threads can take: by several launches that cover them."""
    rc, made = launches(entry, dtype, out_dtype, rows, rows, hidden)
    assert fits(rc, made) and len(made) == parts
    assert sum(m.grid[0] * m.threads for m in made) >= rows * (16 if hidden == 1 else 256)


def test_fp32_rows_past_a_grid(launches):
    """A thread stores half as many fp32 values: 256 threads a row from 1025 columns."""
    rc, made = launches(DEQUANTISE, F32, 0, 1 << 24, 1, 1025)
    assert fits(rc, made) and len(made) == 2


@pytest.mark.parametrize("vocab,hidden,dtype", [((1 << 30) + 1, 8, F32), ((1 << 31) - 1, 4, F32), ((1 << 31) - 1, 64, BF16)])
@pytest.mark.parametrize("n", [1, 900, 20000])
def test_gradients_of_huge_vocabularies(launches, n, vocab, hidden, dtype):
    """The sort's workgroups (one to 1024 ids) and those of the zeros beside them in one grid."""
    rc, made = launches(GRADIENT, BF16, dtype, n, vocab, hidden)
    assert fits(rc, made) and made[0].grid[0] > 1 << 21


def test_gradients_of_more_tiles_than_a_grid(launches):
    """Sizes past it are refused before any launch."""
    assert launches(GRADIENT, BF16, F32, 1 << 30, 1000, 16 * 2048 + 1) == (1, [])


def test_gpu_cases_reach_every_tile_shape(launches):
    """The kernels that some call can launch are those that the GPU tests' cases launch."""
    import torch
    from tests.test_gpu_mx4head import COLUMNS, SHAPES
    code = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, "mx4": MX4}

    def kernel(M, V, dtype, out_dtype):
        rc, made = launches(HEAD, dtype, out_dtype, M, V, COLUMNS[torch.float32])
        assert fits(rc, made) and len(made) == 1
        return made[0].kernel
    tested = {kernel(M, V, code[d], code[o]) for M, V, d in SHAPES for o in COLUMNS}
    reached = {kernel(M, V, d, o) for d in (BF16, F16, MX4) for o in (F32, BF16, F16)
               for M in (1, 9, 17, 33, 65, 129, 257, 2000) for V in (1, 16601, 22001, 151936)}
    assert reached == tested and len(tested) == len(SHAPES) * len(COLUMNS)
