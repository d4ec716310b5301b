"""The vocabulary table's kernels under host sanitizers (CPU, no GPU): the
quantiser, the row gather and the gradient's sort, tiles and join, compiled
unchanged for x86 over the HIP emulation (``tests/hostemu``).  Every array is a
heap allocation of exactly its size, so an access past it stops the run; a run
that finishes must also give the operators' results."""

import hashlib
import os
import shutil
import struct
import subprocess

import numpy as np
import pytest
import torch

from tests import mx4_reference as R
from tests.test_hostemu import BUILD, CLANG, CSRC, DT, EMU, REPO, _exec

FILES = ("run_table.cpp", "mx4_ops.h", os.path.join("shim", "hip", "hip_runtime.h"))


@pytest.fixture(scope="session")
def run_table():
    if not os.path.exists(CLANG):
        pytest.skip("no ROCm clang++ for the host build")
    os.makedirs(BUILD, exist_ok=True)
    h = hashlib.sha256()
    for p in [os.path.join(EMU, f) for f in FILES] + [os.path.join(REPO, "include", "lps.h")] + sorted(
            os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".hip"))):
        h.update(open(p, "rb").read())
    exe = os.path.join(BUILD, f"run_table_{h.hexdigest()[:16]}")
    if not os.path.exists(exe):
        for old in os.listdir(BUILD):
            if old.startswith("run_table_") and "." not in old:
                os.remove(os.path.join(BUILD, old))
        cmd = [CLANG, "-std=c++20", "-O0", "-g1", "-ffp-contract=off",
               "-fsanitize=address,undefined", "-fsanitize=bounds", "-fno-sanitize-recover=all",
               "-I", os.path.join(EMU, "shim"), "-I", os.path.join(REPO, "include"), "-I", CSRC,
               "-x", "c++", os.path.join(EMU, "run_table.cpp"), "-o", f"{exe}.{os.getpid()}", "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-4000:]
        shutil.move(f"{exe}.{os.getpid()}", exe)
    return exe


def _bytes(t):
    t = t.contiguous()
    return (t.view(torch.int16) if t.dtype in (torch.bfloat16, torch.float16) else t).numpy().tobytes()


def _run(exe, tmp_path, header, *arrays):
    inp, out = tmp_path / "in.bin", tmp_path / "out.bin"
    with open(inp, "wb") as f:
        f.write(struct.pack("<16i", *header, *[0] * (16 - len(header))))
        for t in arrays:
            f.write(_bytes(t))
    return _exec(exe, inp, out)


def _take(raw, *parts):
    """The typed arrays that raw holds one after another."""
    out, at = [], 0
    for dtype, *shape in parts:
        n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        out.append(torch.frombuffer(bytearray(raw[at:at + n]), dtype=dtype).reshape(shape))
        at += n
    assert at == len(raw)
    return out


def _f32_bits(x):
    return struct.unpack("<i", struct.pack("<f", x))[0]


@pytest.mark.parametrize("dtype,out_dtype,rows,hidden,pad,words", [
    (torch.bfloat16, torch.bfloat16, 3, 128, 0, True),     # whole groups of four blocks
    (torch.float32, torch.float32, 5, 1601, 0, False),     # a block of one value, rows off the 16-byte lines
    (torch.float16, torch.float32, 9, 33, 3, True),        # padded input rows
    (torch.bfloat16, torch.float16, 2, 4203, 5, False),    # more than one step of a row's threads
    (torch.float32, torch.bfloat16, 17, 7, 0, True),       # part of one block
])
def test_quantise(run_table, tmp_path, dtype, out_dtype, rows, hidden, pad, words):
    g = torch.Generator().manual_seed(rows + hidden)
    x = R.hard_values(rows, hidden + pad, dtype, g)
    nb = -(-hidden // 32)
    ss = nb + (-nb % 4 if words else 0)
    flat = x.reshape(-1)[:(rows - 1) * (hidden + pad) + hidden]
    codes, scales, values = _take(
        _run(run_table, tmp_path, (1, DT[dtype], DT[out_dtype], rows, hidden, hidden + pad, ss), flat),
        (torch.uint8, rows, nb * 16), (torch.uint8, (rows - 1) * ss + nb), (out_dtype, rows, hidden))
    c, s = R.quantise(x[:, :hidden])
    scales = torch.cat([scales, torch.full((ss - nb,), 0x5A, dtype=torch.uint8)]).reshape(rows, ss)
    assert torch.equal(codes, c) and torch.equal(scales[:, :nb], s)
    assert bool((scales[:, nb:] == 0x5A).all())            # nothing written past a row's blocks
    want = R.values(c, s, hidden).to(out_dtype)
    assert torch.equal(values.nan_to_num(nan=1e4), want.nan_to_num(nan=1e4))


@pytest.mark.parametrize("table,out_dtype,n,vocab,hidden,id_dtype", [
    ("mx4", torch.bfloat16, 5, 7, 160, torch.int64),
    ("mx4", torch.float32, 3, 5, 4107, torch.int32),
    (torch.bfloat16, torch.bfloat16, 1, 3, 2056, torch.int64),    # one row over two workgroups
    (torch.float32, torch.bfloat16, 19, 11, 1601, torch.int32),
    (torch.float16, torch.float32, 33, 1, 5, torch.int64)])
def test_lookup(run_table, tmp_path, table, out_dtype, n, vocab, hidden, id_dtype):
    g = torch.Generator().manual_seed(n + hidden)
    w = torch.randn((vocab, hidden), generator=g).to(torch.bfloat16 if table == "mx4" else table)
    ids = torch.randint(-2, vocab + 2, (n,), generator=g).to(id_dtype)
    ids[0] = vocab - 1
    if id_dtype == torch.int64 and n > 2:
        ids[1], ids[2] = 2 ** 40 + 1, -2 ** 62             # nothing but the whole number counts
    if table == "mx4":
        arrays = R.quantise(w)
        values = R.values(*arrays, hidden)
    else:
        arrays, values = (w,), w.double()
    code = 3 if table == "mx4" else DT[table]
    (out,) = _take(_run(run_table, tmp_path, (2, code, DT[out_dtype], n, vocab, hidden, ids.element_size(), _f32_bits(1.5)),
                        ids, *arrays), (out_dtype, n, hidden))
    valid = (ids >= 0) & (ids < vocab)
    want = torch.where(valid[:, None], values[torch.where(valid, ids, 0).long()] * 1.5, 0.0).float().to(out_dtype)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,out_dtype,n,vocab,hidden,accumulate,ids_kind", [
    (torch.bfloat16, torch.float32, 70, 30, 40, False, "mixed"),
    (torch.float16, torch.bfloat16, 300, 9, 300, True, "mixed"),      # ids of many positions, two workgroups a row
    (torch.float32, torch.float32, 67, 5, 264, False, "one"),         # one id everywhere
    (torch.float32, torch.float16, 5, 700, 3, False, "distinct"),     # a single id each, rows of zeros
    (torch.bfloat16, torch.float32, 2100, 60, 2057, False, "mixed"), # three launches: runs over many tiles, two workgroups a tile
    (torch.bfloat16, torch.float32, 4500, 3, 8, True, "one"),         # a list that outgrows LDS
    (torch.bfloat16, torch.float32, 6, 4, 16, False, "none"),         # no position counts
    (torch.float32, torch.float32, 1, 1, 1, False, "one"),
    (torch.float32, torch.bfloat16, 0, 33, 9, False, "none")])
def test_gradient(run_table, tmp_path, dtype, out_dtype, n, vocab, hidden, accumulate, ids_kind):
    """Against the sum in 64 bits: fp32 sums of k terms are off by at most (k -
    1) 2^-24 of the sum of magnitudes, then the scale and the store round once each."""
    g = torch.Generator().manual_seed(n + vocab + hidden)
    ids = {"mixed": torch.randint(-1, vocab, (n,), generator=g), "one": torch.full((n,), vocab - 1),
           "distinct": torch.randperm(vocab, generator=g)[:n], "none": torch.full((n,), vocab)}[ids_kind]
    ids = ids.to(torch.int64 if n % 2 else torch.int32)
    grad = torch.randn((n, hidden), generator=g).to(dtype)
    out0 = torch.randn((vocab, hidden), generator=g).to(out_dtype)
    (out,) = _take(_run(run_table, tmp_path, (3, DT[dtype], DT[out_dtype], n, vocab, hidden, ids.element_size(),
                                              _f32_bits(0.75), int(accumulate)), ids, grad, out0), (out_dtype, vocab, hidden))
    want, bound = R.gradient(ids, grad, vocab, 0.75, out0 if accumulate else None, out_dtype)
    assert bool(((out.double() - want).abs() <= bound).all())
    touched = torch.zeros(vocab, dtype=torch.bool)
    touched[ids[(ids >= 0) & (ids < vocab)].long()] = True
    if accumulate:
        assert torch.equal(out[~touched], out0[~touched])
    else:
        assert bool((out[~touched] == 0).all())


HEADS = [(131, 294, torch.bfloat16, torch.bfloat16),      # stages, blocks and a part of one
         (130, 40, torch.float16, torch.float32),         # less than a stage
         (140, 1061, torch.float16, torch.bfloat16),      # more stages than buffers
         (258, 768, "mx4", torch.bfloat16),               # whole stages
         (129, 163, "mx4", torch.float32)]                # a stage and parts of blocks


@pytest.mark.parametrize("M,V,H,dtype,out_dtype", [(M, *c) for c in HEADS for M in (1, 13, 33, 70)] +
                         [(257, *HEADS[4])])
def test_head(run_table, tmp_path, monkeypatch, M, V, H, dtype, out_dtype):
    """Every tile shape: in bounds; logits within one rounding of the output type
    and the fp32 accumulation (H 2^-24 of the sum of magnitudes), block maxima
    exact, sums within 2e-6."""
    monkeypatch.setenv("LPS_EMU_CUS", "1")     # no grid's tiles all run at once: the shapes go by the rows
    g = torch.Generator().manual_seed(M + V + H)
    x = torch.randn((M, H), generator=g).to(torch.bfloat16 if dtype == "mx4" else dtype)
    w = (torch.randn((V, H), generator=g) * (2.0 / H ** 0.5)).to(torch.bfloat16)
    c, s = R.quantise(w)
    if dtype == torch.float16:
        s[5, 0], s[77, 1], s[9] = 255, 90, 150       # NaN, and scales past fp16's exponents
        c[77] = 0x22
        x[0, 0] = float("inf")
        x[M // 2, 1] = 6e-8
    nb = -(-H // 32)
    ss = nb + -nb % 4
    pad = lambda t: torch.cat([t, torch.full((t.shape[0], ss - nb), 255, dtype=torch.uint8)], 1).reshape(-1)[:(t.shape[0] - 1) * ss + nb]  # noqa: E731
    xs = H + -H % 8
    if dtype == "mx4":
        xc, xsc = R.quantise(x)
        arrays, xv = (xc, pad(xsc)), R.values(xc, xsc, H)
    else:
        wide = torch.full((M, xs), float("nan"), dtype=dtype)
        wide[:, :H] = x
        arrays, xv = (wide.reshape(-1)[:(M - 1) * xs + H],), x.double()
    if H % 32:
        c[:, -1] |= 0x70                              # codes past the row's end: nothing they hold counts
    G = -(-V // 128)
    out, st = _take(_run(run_table, tmp_path, (4, 3 if dtype == "mx4" else DT[dtype], DT[out_dtype], M, V, H, xs, ss),
                         *arrays, c, pad(s)), (out_dtype, M, V), (torch.float32, M, G, 2))
    wv = R.values(c, s, H)
    ref, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    out, st = out.double(), st.double()
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(out)) and torch.equal(torch.isnan(ref), torch.isnan(out))
    assert torch.equal(ref[~fine].nan_to_num(nan=1.0), out[~fine].nan_to_num(nan=1.0))
    err = (out - ref).abs()[fine]
    assert bool((err <= R.HALF[out_dtype][0] * ref.abs()[fine] * 1.01 + H * 2.0 ** -24 * mag[fine]).all())
    if dtype != torch.float16:
        blocks = torch.cat([out, torch.full((M, G * 128 - V), float("-inf"), dtype=torch.float64)], 1).reshape(M, G, 128)
        mx = blocks.max(dim=2).values
        assert torch.equal(st[..., 0], mx)
        torch.testing.assert_close(st[..., 1], torch.exp(blocks - mx.unsqueeze(-1)).sum(dim=2), rtol=2e-6, atol=0)


@pytest.mark.parametrize("M", [3, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_weights_past_fp32(run_table, tmp_path, monkeypatch, M, dtype):
    """Scale bytes 253 and 254, which the quantiser never gives, hold values past
    fp32's largest: infinities to 16-bit states, as to the dequantiser, whatever else
    the row holds and however a state is taken apart."""
    monkeypatch.setenv("LPS_EMU_CUS", "1")
    V, H = 130, 290
    c, s, x = R.extreme_scales(V, H, M, dtype)
    nb, xs = s.shape[1], H + -H % 8
    ss = nb + -nb % 4
    pad = torch.cat([s, torch.full((V, ss - nb), 255, dtype=torch.uint8)], 1).reshape(-1)[:(V - 1) * ss + nb]
    wide = torch.zeros((M, xs), dtype=dtype)
    wide[:, :H] = x
    out, _ = _take(_run(run_table, tmp_path, (4, DT[dtype], DT[torch.float32], M, V, H, xs, ss),
                        wide.reshape(-1)[:(M - 1) * xs + H], c, pad), (torch.float32, M, V), (torch.float32, M, 2, 2))
    R.check_extreme(out, R.extreme_products(c, s, x))
