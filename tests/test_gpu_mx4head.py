"""The LM head over a 4-bit weight (``lm_head`` with an ``Mx4Tensor``) on the
GPU, against the products in 64 bits.

Bound: one rounding of the output type, and the fp32 accumulation of H exact
products: H 2^-24 of the sum of magnitudes."""

import pytest
import torch

import lps
from tests import mx4_reference as R

pytestmark = pytest.mark.gpu


def _weight(V, H, g, deviation=2.0):
    """A 4-bit weight on the CPU: (codes, scales, values in 64 bits)."""
    c, s = R.quantise((torch.randn((V, H), generator=g) * (deviation / H ** 0.5)).bfloat16())
    return c, s, R.values(c, s, H)


def _check(out, x, w, H):
    ref, mag = x @ w.T, x.abs() @ w.abs().T
    err = (out.double().cpu() - ref).abs()
    half, least = R.HALF[out.dtype]
    bound = half * 1.01 * ref.abs() + H * 2.0 ** -24 * mag + least
    assert bool((err <= bound).all()), f"past the bound by {float((err - bound).max())}"


def _check_stats(out, stats):
    M, V = out.shape
    G = -(-V // 128)
    v = torch.cat([out.double().cpu(), torch.full((M, G * 128 - V), float("-inf"), dtype=torch.float64)], 1).reshape(M, G, 128)
    mx = v.amax(2)
    assert torch.equal(stats[..., 0].double().cpu(), mx)
    torch.testing.assert_close(stats[..., 1].double().cpu(), torch.exp(v - mx.unsqueeze(-1)).sum(2), rtol=2e-6, atol=0)


@pytest.mark.parametrize("M", [1, 2, 31, 32, 33, 64, 65, 96, 97, 128, 129, 256, 257, 513])
@pytest.mark.parametrize("V,H,dtype,out_dtype", [
    (301, 1601, torch.bfloat16, torch.bfloat16),     # odd everywhere
    (640, 1024, torch.float16, torch.float32),       # whole stages
    (260, 96, torch.bfloat16, torch.float32),        # fewer stages than buffers
    (129, 7, torch.float16, torch.float16),          # part of a block
    (771, 1100, "mx4", torch.bfloat16),
    (512, 2048, "mx4", torch.float32),
    (1, 33, "mx4", torch.float16)])
def test_head(dev, M, V, H, dtype, out_dtype):
    g = torch.Generator().manual_seed(M * 11 + V + H)
    c, s, w = _weight(V, H, g)
    x = torch.randn((M, H), generator=g).to(torch.bfloat16 if dtype == "mx4" else dtype)
    if dtype == "mx4":
        arg = lps.mx4_quantize(x.to(dev))
        xv = R.values(*R.quantise(x), H)
    else:
        arg, xv = x.to(dev), x.double()
    out, stats = lps.lm_head(arg, lps.Mx4Tensor(c.to(dev), s.to(dev), H), out_dtype=out_dtype, return_stats=True)
    assert out.dtype == out_dtype and out.shape == (M, V)
    _check(out, xv, w, H)
    _check_stats(out, stats)


def test_head_quantised_here(dev):
    """The weight from mx4_quantize, default output types, leading dimensions."""
    g = torch.Generator().manual_seed(1)
    w = (torch.randn((700, 416), generator=g) * 0.1).bfloat16()
    x = torch.randn((2, 3, 416), generator=g).half()
    t = lps.mx4_quantize(w.to(dev))
    out = lps.lm_head(x.to(dev), t)
    assert out.dtype == torch.float16 and out.shape == (2, 3, 700)
    _check(out.reshape(6, 700), x.reshape(6, 416).double(), R.values(*R.quantise(w), 416), 416)
    assert lps.lm_head(lps.mx4_quantize(x.to(dev)), t).dtype == torch.bfloat16
    assert lps.lm_head(x[:, :0].to(dev), t).shape == (2, 0, 700)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, "mx4"])
@pytest.mark.parametrize("M", [5, 70, 300])
def test_head_strides_and_guards(dev, dtype, M):
    """Operands inside wider buffers (whose other bytes are NaN codes and scales), at every alignment."""
    g = torch.Generator().manual_seed(M)
    V, H = 301, 230
    c, s, w = _weight(V, H, g)
    nb = s.shape[1]
    x = torch.randn((M, H), generator=g).to(torch.bfloat16 if dtype == "mx4" else dtype)
    for off in (0, 1, 4):
        wide_c = torch.full((V, 16 * nb + 48), 0x77, dtype=torch.uint8, device=dev)
        wide_s = torch.full((V, nb + 9), 255, dtype=torch.uint8, device=dev)
        wc, wsc = wide_c[:, 16 * (off % 3):][:, :16 * nb], wide_s[:, off:off + nb]
        wc.copy_(c), wsc.copy_(s)
        if dtype == "mx4":
            xc, xs = R.quantise(x)
            xw = torch.full((M, nb + 3), 255, dtype=torch.uint8, device=dev)
            xw[:, off % 3:off % 3 + nb] = xs.to(dev)
            arg, xv = lps.Mx4Tensor(xc.to(dev), xw[:, off % 3:off % 3 + nb], H), R.values(xc, xs, H)
        else:
            xw = torch.full((M, H + 18), float("nan"), dtype=dtype, device=dev)
            xw[:, off:off + H] = x.to(dev)
            arg, xv = xw[:, off:off + H], x.double()
        _check(lps.lm_head(arg, lps.Mx4Tensor(wc, wsc, H), out_dtype=torch.float32), xv, w, H)


@pytest.mark.parametrize("M", [3, 150])
def test_head_far_scales_of_fp16(dev, M):
    """fp16 hidden states against scales outside fp16's exponents, one row of
    each: products that are all of the answer there."""
    g = torch.Generator().manual_seed(M)
    V, H = 256, 416
    codes = torch.randint(0, 256, (V, 208), generator=g).to(torch.uint8)
    scales = torch.arange(1, 257).clamp(max=200).to(torch.uint8).unsqueeze(1).repeat(1, 13)
    scales[::5, 3] = 120
    x = (torch.randn((M, H), generator=g) * 2.0 ** torch.randint(-14, 4, (M, H), generator=g).float()).half()
    out = lps.lm_head(x.to(dev), lps.Mx4Tensor(codes.to(dev), scales.to(dev), H), out_dtype=torch.float32)
    w = R.values(codes, scales, H)
    # (products under fp32's normal range are not kept to their last bit)
    ref, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    assert bool(((out.double().cpu() - ref).abs() <= 2.0 ** -24 * 1.01 * ref.abs() + H * 2.0 ** -24 * mag + H * 2.0 ** -126).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, "mx4"])
def test_head_values_that_are_not_finite(dev, dtype):
    """A NaN block makes its column NaN, an infinity or NaN in x its row what the products say."""
    g = torch.Generator().manual_seed(4)
    M, V, H = 40, 200, 300
    c, s, w = _weight(V, H, g)
    s[17, 2] = 255
    w = R.values(c, s, H)
    x = torch.randn((M, H), generator=g).to(torch.bfloat16 if dtype == "mx4" else dtype)
    x[3, 5], x[7, 299], x[8, 0] = float("nan"), float("inf"), float("-inf")
    if dtype == "mx4":
        arg, xv = lps.mx4_quantize(x.to(dev)), R.values(*R.quantise(x), H)
    else:
        arg, xv = x.to(dev), x.double()
    out = lps.lm_head(arg, lps.Mx4Tensor(c.to(dev), s.to(dev), H), out_dtype=torch.float32).double().cpu()
    ref = xv @ w.T
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isinf(), ref.isinf())
    assert torch.equal(out[ref.isinf()], ref[ref.isinf()])
    fine = ref.isfinite()
    mag = xv.abs() @ w.abs().T
    assert bool(((out - ref).abs()[fine] <= (2.0 ** -24 * 1.01 * ref.abs() + H * 2.0 ** -24 * mag)[fine]).all())


@pytest.mark.parametrize("dtype,M", [(torch.bfloat16, 64), (torch.float16, 1), ("mx4", 200)])
def test_head_real_size(dev, dtype, M):
    """A decode batch at 4096 -> 151936, against the products in fp64 on the GPU; equal calls give equal bits."""
    g = torch.Generator(device=dev).manual_seed(6)
    V, H = 151936, 4096
    t = lps.mx4_quantize(torch.randn((V, H), generator=g, device=dev, dtype=torch.bfloat16) * 0.04)
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16 if dtype == "mx4" else dtype)
    arg = lps.mx4_quantize(x) if dtype == "mx4" else x
    xv = lps.mx4_dequantize(arg, torch.float32).double() if dtype == "mx4" else x.double()
    out = lps.lm_head(arg, t)
    assert torch.equal(out, lps.lm_head(arg, t))
    w = lps.mx4_dequantize(t, torch.float32).double()
    ref, mag = xv @ w.T, xv.abs() @ w.abs().T
    half, least = R.HALF[out.dtype]
    assert bool(((out.double() - ref).abs() <= half * 1.01 * ref.abs() + H * 2.0 ** -24 * mag + least).all())


def test_decode_step(dev):
    """The table at both ends of a decode step, captured: lookup, head with
    statistics, softmax; replays give the eager results."""
    g = torch.Generator().manual_seed(9)
    V, H, B = 5003, 384, 6
    t = lps.mx4_quantize((torch.randn((V, H), generator=g) * 0.3).bfloat16().to(dev))
    ids = torch.zeros((B,), dtype=torch.int64, device=dev)

    def step():
        h = lps.embedding(ids, t, scale=2.0)
        logits, stats = lps.lm_head(h, t, return_stats=True)
        return h, logits, lps.fused_softmax(logits, row_stats=stats)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        ids.copy_(torch.randint(-1, V, (B,), generator=g))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals(dev):
    t = lps.mx4_quantize(torch.zeros((8, 64), device=dev))
    x = torch.zeros((2, 64), device=dev, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        lps.lm_head(x.float(), t)
    with pytest.raises(TypeError):
        lps.lm_head(lps.mx4_quantize(x), x)
    with pytest.raises(ValueError):
        lps.lm_head(x[:, :63], t)
    with pytest.raises(TypeError):
        lps.lm_head(x, t, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        lps.lm_head(x, lps.Mx4Tensor(t.codes, t.scales[:4], 64))
    with pytest.raises(TypeError):
        lps.lm_head(x, lps.Mx4Tensor(t.codes.int(), t.scales, 64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        lps.lm_head(x.cpu(), t)


@pytest.mark.parametrize("M,H,xs,dtype", [
    (3, (1 << 22) + 8, (1 << 22) + 8, torch.float16), (2, (1 << 22) + 3, (1 << 22) + 3, torch.bfloat16),
    (1, 1 << 24, 1 << 24, torch.bfloat16), (2, 1 << 24, 1 << 23, "mx4"), (5, 96, (1 << 22) + 8, torch.bfloat16),
    (5, 96, (1 << 23) + 16, "mx4")])
def test_head_rows_far_apart(dev, M, H, xs, dtype):
    """Long rows and rows more than 8 MiB apart: sums of whole numbers, the same bits as in 64."""
    g = torch.Generator().manual_seed(M + H)
    V, n = 3, -(-H // 32)
    codes = torch.randint(0, 256, (V, 16 * n), generator=g).to(torch.uint8)
    scales = torch.full((V, n), 128, dtype=torch.uint8)               # values of -12 .. 12
    wide = torch.zeros((V, (1 << 23) + 16), dtype=torch.uint8, device=dev)
    wide[:, :16 * n] = codes.to(dev)
    at = torch.randint(0, H, (M, 500), generator=g)
    at[:, 0], at[:, 1] = H - 1, 0
    x = torch.zeros((M, H)).scatter_(1, at, torch.randint(1, 3, (M, 500), generator=g).float())
    if dtype == "mx4":
        c, s = R.quantise(x)
        rows = torch.zeros(((M - 1) * xs + 16 * n,), dtype=torch.uint8, device=dev).as_strided((M, 16 * n), (xs, 1))
        arg = lps.Mx4Tensor(rows.copy_(c), s.to(dev), H)
    else:
        arg = torch.zeros(((M - 1) * xs + H,), dtype=dtype, device=dev).as_strided((M, H), (xs, 1)).copy_(x)
    out, stats = lps.lm_head(arg, lps.Mx4Tensor(wide[:, :16 * n], scales.to(dev), H), out_dtype=torch.float32, return_stats=True)
    ref = torch.stack([x.double() @ R.values(codes[v:v + 1], scales[v:v + 1], H)[0] for v in range(V)], 1)
    assert torch.equal(out.double().cpu(), ref)
    assert torch.equal(stats[..., 0].double().cpu(), ref.amax(1, keepdim=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,H", [(3, 290), (70, 290), (20, 1024)])
def test_head_weights_past_fp32(dev, dtype, M, H):
    """The largest and the smallest scale bytes: values past fp32's range are
    infinities to 16-bit states, as to the dequantiser."""
    V = 517
    c, s, x = R.extreme_scales(V, H, M, dtype)
    t = lps.Mx4Tensor(c.to(dev), s.to(dev), H)
    assert torch.equal(lps.mx4_dequantize(t, torch.float32).cpu(), R.values(c, s, H).float())
    R.check_extreme(lps.lm_head(x.to(dev), t, out_dtype=torch.float32), R.extreme_products(c, s, x))


# (rows, vocab, states' type) such that each tile shape is taken on 256 CUs: a grid that
# runs at once takes the smallest tiles, so the larger ones need many columns.
SHAPES = ([(M, V, d) for d in (torch.bfloat16, torch.float16)
           for M, V in ((7, 301), (16, 301), (31, 301), (64, 32897), (130, 22001))] +
          [(30, 301, "mx4"), (64, 16601, "mx4"), (128, 16601, "mx4"), (300, 22001, "mx4")])
# part of a block after whole stages; whole stages; a block and a part after more stages than the rings hold
COLUMNS = {torch.float32: 1380, torch.bfloat16: 2048, torch.float16: 4139}


@pytest.mark.parametrize("out_dtype", list(COLUMNS))
@pytest.mark.parametrize("M,V,dtype", SHAPES)
def test_every_tile_shape(dev, M, V, dtype, out_dtype):
    """Each kernel at an odd vocabulary, against the products in fp64 on the GPU, with
    block statistics; of fp16, rows whose scales it does not hold."""
    H = COLUMNS[out_dtype]
    g = torch.Generator(device=dev).manual_seed(M + V + H)
    t = lps.mx4_quantize((torch.randn((V, H), generator=g, device=dev) * (2.0 / H ** 0.5)).bfloat16())
    far = dtype == torch.float16
    if far:                  # tiny, and where no sum of exponentials is compared huge
        t.scales[::5, 3:9] -= 20
        if out_dtype == torch.float32:
            t.scales[1::5] += 25
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16 if dtype == "mx4" else dtype)
    arg = lps.mx4_quantize(x) if dtype == "mx4" else x
    out, stats = lps.lm_head(arg, t, out_dtype=out_dtype, return_stats=True)
    again, again_stats = lps.lm_head(arg, t, out_dtype=out_dtype, return_stats=True)
    assert torch.equal(out, again) and torch.equal(stats, again_stats)
    xv = lps.mx4_dequantize(arg, torch.float32).double() if dtype == "mx4" else x.double()
    w = lps.mx4_dequantize(t, torch.float32).double()
    ref, mag = xv @ w.T, xv.abs() @ w.abs().T
    half, least = R.HALF[out_dtype]
    off = (out.double() - ref).abs() - (half * 1.01 * ref.abs() + H * 2.0 ** -24 * mag + least)
    assert bool((off <= 0).all()), f"past the bound by {float(off.max())}"
    if far and out_dtype == torch.float32:
        blocks = torch.cat([out, torch.full((M, -V % 128), float("-inf"), device=dev)], 1).reshape(M, -1, 128)
        assert torch.equal(stats[..., 0], blocks.amax(2))
    else:
        _check_stats(out, stats)
