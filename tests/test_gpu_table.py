"""The vocabulary table's operators on the GPU: microscaled 4-bit quantisation,
the embedding lookup and its gradient, against their definitions in 64 bits."""

import pytest
import torch

import lps
from tests import mx4_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---------------------------------------------------------------- quantiser --


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (6, 32), (7, 33), (129, 1601), (9, 4096), (3, 4107), (5, 16384), (300, 40)])
def test_quantise(dev, dtype, rows, hidden):
    """Codes and scales are the definition's; so are the values of every type."""
    g = torch.Generator().manual_seed(rows * 31 + hidden)
    x = R.hard_values(rows, hidden, dtype, g)
    t = lps.mx4_quantize(x.to(dev))
    c, s = R.quantise(x)
    assert torch.equal(t.codes.cpu(), c) and torch.equal(t.scales.cpu(), s)
    for out_dtype in DTYPES:
        v = lps.mx4_dequantize(t, out_dtype)
        want = R.values(c, s, hidden).to(out_dtype)
        assert v.dtype == out_dtype and torch.equal(v.cpu().nan_to_num(nan=3e4), want.nan_to_num(nan=3e4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_every_16_bit_value(dev, dtype):
    """Every value under its own scale and under those of larger neighbours."""
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    x = torch.zeros((v.numel(), 32 * 5), dtype=dtype)
    for k in range(5):
        x[:, 32 * k + 3] = v
        big = (v.double().abs() * 2.0 ** k).clamp(max=torch.finfo(dtype).max)
        x[:, 32 * k + 17] = big.to(dtype)
    t = lps.mx4_quantize(x.to(dev))
    c, s = R.quantise(x)
    assert torch.equal(t.codes.cpu(), c) and torch.equal(t.scales.cpu(), s)


def test_quantise_shapes_and_strides(dev):
    g = torch.Generator().manual_seed(2)
    x = torch.randn((3, 4, 70), generator=g)
    for y in (x.to(dev), x.to(dev)[:, :, :65], x.to(dev).transpose(0, 1), x.to(dev)[0], x.to(dev)[1, 2],
              x.to(dev)[:1].expand(5, 4, 70), torch.empty((0, 70), device=dev)):
        t = lps.mx4_quantize(y)
        n = -(-y.shape[-1] // 32)
        assert t.shape == y.shape and t.codes.shape == (*y.shape[:-1], 16 * n) and t.scales.shape == (*y.shape[:-1], n)
        c, s = R.quantise(y.cpu().reshape(-1, y.shape[-1]))
        assert torch.equal(t.codes.cpu().reshape(c.shape), c) and torch.equal(t.scales.cpu().reshape(s.shape), s)
        assert torch.equal(lps.mx4_dequantize(t, torch.float32).cpu().reshape(-1, y.shape[-1]),
                           R.values(c, s, y.shape[-1]).float())


def test_dequantise_any_scale(dev):
    """Tables from elsewhere: every scale byte, 0 (2^-127) and 255 (NaN) among them."""
    codes = torch.arange(256, dtype=torch.uint8).reshape(16, 16).repeat(16, 1)
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    for dtype in DTYPES:
        v = lps.mx4_dequantize(lps.Mx4Tensor(codes.to(dev), scales.to(dev), 32), dtype)
        want = R.values(codes, scales, 32).to(dtype)
        assert torch.equal(v.cpu().nan_to_num(nan=1.25), want.nan_to_num(nan=1.25))


# ------------------------------------------------------------------- lookup --


@pytest.mark.parametrize("table", ["mx4"] + DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,hidden", [(1, 50, 4096), (2, 1, 1), (160, 517, 1601), (300, 129, 72), (5000, 1000, 512)])
def test_lookup(dev, table, out_dtype, n, vocab, hidden):
    """One product in fp32 and one rounding: the same bits as there."""
    g = torch.Generator().manual_seed(n + vocab + hidden)
    w = torch.randn((vocab, hidden), generator=g).to(torch.bfloat16 if table == "mx4" else table)
    ids = torch.randint(-2, vocab + 2, (n,), generator=g)
    ids[-1] = vocab - 1
    if table == "mx4":
        c, s = R.quantise(w)
        arg, values = lps.Mx4Tensor(c.to(dev), s.to(dev), hidden), R.values(c, s, hidden).float()
    else:
        arg, values = w.to(dev), w.float()
    valid = (ids >= 0) & (ids < vocab)
    want = torch.where(valid[:, None], values[torch.where(valid, ids, 0)] * torch.tensor(hidden ** 0.5), 0.0).to(out_dtype)
    for i in (ids, ids.to(torch.int32)):
        out = lps.embedding(i.to(dev), arg, scale=hidden ** 0.5, out_dtype=out_dtype)
        assert out.dtype == out_dtype and torch.equal(out.cpu(), want)


def test_lookup_shapes_strides_and_far_ids(dev):
    g = torch.Generator().manual_seed(3)
    w = torch.randn((40, 100), generator=g)
    ids = torch.tensor([[1, -1, 39], [2 ** 32 + 1, 0, -2 ** 63]])
    want = torch.where(((ids >= 0) & (ids < 40))[..., None], w[torch.where((ids >= 0) & (ids < 40), ids, 0)], 0.0)
    assert torch.equal(lps.embedding(ids.to(dev), w.to(dev)).cpu(), want)
    assert torch.equal(lps.embedding(ids.to(dev).t(), w.to(dev)).cpu(), want.transpose(0, 1))
    wide = torch.randn((40, 137), generator=g).to(dev)
    wide[:, 5:105] = w.to(dev)
    assert torch.equal(lps.embedding(ids.to(dev), wide[:, 5:105]).cpu(), want)      # rows of a wider buffer, off 16 bytes
    assert torch.equal(lps.embedding(ids.to(dev), w.t().contiguous().to(dev).t()).cpu(), want)
    assert lps.embedding(torch.empty((2, 0), dtype=torch.int64, device=dev), w.to(dev)).shape == (2, 0, 100)
    assert torch.equal(lps.embedding(ids[0, 0].to(dev), w.to(dev)).cpu(), w[1])
    # rows that hold infinities and NaN do not reach positions without a token
    bad = torch.full((40, 100), float("nan"))
    assert bool((lps.embedding(torch.full((3,), -1, device=dev), bad.to(dev)) == 0).all())


def test_lookup_past_32_bits(dev):
    """A table of more than 2^32 bytes (and elements): its last rows."""
    vocab, hidden = 540000, 8192
    w = torch.zeros((vocab, hidden), dtype=torch.bfloat16, device=dev)
    w[-3:] = torch.arange(3 * 64, device=dev).reshape(3, 64).repeat(1, 128).to(torch.bfloat16)
    out = lps.embedding(torch.tensor([vocab - 3, vocab - 1, vocab], device=dev), w)
    assert torch.equal(out[:2], w[[-3, -1]]) and bool((out[2] == 0).all())


# ----------------------------------------------------------------- gradient --


def _ids(kind, n, vocab, g):
    if kind == "one":
        return torch.full((n,), vocab // 2)
    if kind == "distinct":
        return torch.randperm(vocab, generator=g)[:n]
    if kind == "text":     # the few frequent ids repeat
        return (vocab ** torch.rand((n,), generator=g, dtype=torch.float64)).long().clamp(max=vocab) - 1
    return torch.randint(-3, vocab + 3, (n,), generator=g)


@pytest.mark.parametrize("kind", ["text", "one", "distinct", "mixed"])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                             (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("n,vocab,hidden", [(1, 1, 1), (17, 40, 33), (517, 1601, 1001), (3000, 32000, 260), (9000, 9001, 72)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(dev, kind, dtype, out_dtype, n, vocab, hidden, accumulate):
    g = torch.Generator().manual_seed(n + vocab + hidden)
    ids = _ids(kind, n, vocab, g)
    n = ids.numel()
    grad = torch.randn((n, hidden), generator=g).to(dtype)
    out0 = torch.randn((vocab, hidden), generator=g).to(out_dtype) if accumulate else None
    want, bound = R.gradient(ids, grad, vocab, 1.7, out0, out_dtype)
    buf = out0.to(dev) if accumulate else None
    got = lps.embedding_grad(ids.to(dev), grad.to(dev), vocab, scale=1.7, out=buf,
                             dtype=None if accumulate else out_dtype)
    assert got.dtype == out_dtype and (got is buf or not accumulate)
    off = (got.double().cpu() - want).abs() - bound
    assert bool((off <= 0).all()), f"past the bound by {float(off.max())}"
    touched = torch.zeros(vocab, dtype=torch.bool)
    touched[ids[(ids >= 0) & (ids < vocab)]] = True
    rest = got.cpu()[~touched]
    assert torch.equal(rest, out0[~touched]) if accumulate else bool((rest == 0).all())
    # the same call again: the same bits
    again = lps.embedding_grad(ids.to(dev).int(), grad.to(dev), vocab, scale=1.7,
                               out=out0.to(dev) if accumulate else None, dtype=None if accumulate else out_dtype)
    assert torch.equal(got, again)


def test_gradient_long_list_of_one_id(dev):
    """70000 positions, most of one id: a list past LDS, a run over hundreds of tiles."""
    g = torch.Generator().manual_seed(8)
    ids = torch.where(torch.rand((70000,), generator=g) < 0.9, 3, torch.randint(0, 50, (70000,), generator=g))
    grad = torch.randn((70000, 24), generator=g)
    want, bound = R.gradient(ids, grad, 50, 1.0, None, torch.float32)
    got = lps.embedding_grad(ids.to(dev), grad.to(dev), 50)
    assert bool(((got.double().cpu() - want).abs() <= bound).all())


def test_gradient_shapes_strides_and_empty(dev):
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, 20, (3, 5), generator=g)
    grad = torch.randn((3, 5, 40), generator=g)
    want, bound = R.gradient(ids.reshape(-1), grad.reshape(15, 40), 20, 1.0, None, torch.float32)
    ok = lambda t: bool(((t.double().cpu() - want).abs() <= bound).all())  # noqa: E731
    assert ok(lps.embedding_grad(ids.to(dev), grad.to(dev), 20))
    wide = torch.randn((3, 5, 63), generator=g).to(dev)
    wide[..., 7:47] = grad.to(dev)
    assert ok(lps.embedding_grad(ids.to(dev), wide[..., 7:47], 20))
    assert ok(lps.embedding_grad(ids.to(dev).t().contiguous().t(), grad.to(dev).transpose(0, 1).contiguous().transpose(0, 1), 20))
    # rows of a wider buffer: nothing beside them is written
    buf = torch.full((20, 50), 7.0, device=dev)
    buf[:, 3:43] = 0.0
    assert ok(lps.embedding_grad(ids.to(dev), grad.to(dev), 20, out=buf[:, 3:43]))
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 43:] == 7).all())
    none = torch.empty((0,), dtype=torch.int64, device=dev)
    assert bool((lps.embedding_grad(none, torch.empty((0, 8), device=dev), 4) == 0).all())
    assert bool((lps.embedding_grad(none, torch.empty((0, 8), device=dev), 4, out=torch.ones((4, 8), device=dev)) == 1).all())
    # a broadcast gradient (of a sum) and one whose values are not finite at missing tokens
    one = torch.ones((1, 40), device=dev).expand(15, 40)
    got = lps.embedding_grad(ids.reshape(-1).to(dev), one, 20)
    assert torch.equal(got[:, 0].cpu(), torch.bincount(ids.reshape(-1), minlength=20).float())
    bad = torch.full((2, 8), float("nan"), device=dev)
    assert bool((lps.embedding_grad(torch.tensor([-1, 4], device=dev), bad, 4) == 0).all())


def test_lookup_backward(dev):
    """Autograd's gradient: against the formula's, and against differences of the
    loss (central, step 2^-6 of fp32 values near 1: the loss is linear in the
    table, so a difference is off by its fp32 roundings alone)."""
    g = torch.Generator().manual_seed(10)
    ids = torch.randint(-1, 12, (2, 9), generator=g)
    w = torch.randn((12, 20), generator=g)
    cot = torch.randn((2, 9, 20), generator=g)
    t = w.to(dev).requires_grad_()
    lps.embedding(ids.to(dev), t, scale=2.0).backward(cot.to(dev))
    want, bound = R.gradient(ids.reshape(-1), cot.reshape(18, 20), 12, 2.0, None, torch.float32)
    assert bool(((t.grad.double().cpu() - want).abs() <= bound).all())
    loss = lambda x: (lps.embedding(ids.to(dev), x, scale=2.0).double() * cot.to(dev).double()).sum()  # noqa: E731
    h = 2.0 ** -6
    for v, c in [(0, 0), (5, 7), (11, 19), (3, 11)]:
        d = torch.zeros_like(w)
        d[v, c] = h
        up, down = loss((w + d).to(dev)), loss((w - d).to(dev))
        # w +- h and 2 (w +- h) are rounded (2^-24 of at most 8), times the 18 gradients' sizes
        noise = 2 * 2.0 ** -24 * 16 * float(cot.abs().sum(dim=(0, 1)).max()) / (2 * h)
        assert abs(float(up - down) / (2 * h) - float(t.grad[v, c])) <= noise
    # a broadcast cotangent, a 16-bit table, a gradient that is added up
    t16 = w.to(dev).bfloat16().requires_grad_()
    lps.embedding(ids.to(dev), t16).sum().backward()
    lps.embedding(ids.to(dev), t16).sum().backward()
    count = torch.bincount(ids[ids >= 0], minlength=12)
    assert t16.grad.dtype == torch.bfloat16 and torch.equal(t16.grad[:, 0].cpu(), (2 * count).bfloat16())


def test_on_another_stream(dev):
    """Calls run on the current stream, workspaces and outputs with them."""
    g = torch.Generator().manual_seed(12)
    w, grad = torch.randn((500, 256), generator=g).to(dev), torch.randn((2000, 256), generator=g).to(dev)
    ids = torch.randint(0, 500, (2000,), generator=g).to(dev)
    a, b, c = lps.embedding(ids, w), lps.embedding_grad(ids, grad, 500), lps.mx4_quantize(w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(5):
            a2, b2, c2 = lps.embedding(ids, w), lps.embedding_grad(ids, grad, 500), lps.mx4_quantize(w)
    s.synchronize()
    assert torch.equal(a, a2) and torch.equal(b, b2) and torch.equal(c.codes, c2.codes) and torch.equal(c.scales, c2.scales)


def test_in_a_graph(dev):
    """Captured once, replayed with eager work between: every replay is the eager result."""
    g = torch.Generator().manual_seed(13)
    w = torch.randn((300, 128), generator=g).to(dev)
    ids, grad = torch.zeros((400,), dtype=torch.int64, device=dev), torch.zeros((400, 128), device=dev)
    lps.embedding(ids, w), lps.embedding_grad(ids, grad, 300), lps.mx4_quantize(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b, c = lps.embedding(ids, w), lps.embedding_grad(ids, grad, 300), lps.mx4_quantize(grad)
    for _ in range(4):
        ids.copy_(torch.randint(-1, 300, (400,), generator=g))
        grad.copy_(torch.randn((400, 128), generator=g))
        graph.replay()
        ea, eb, ec = lps.embedding(ids, w), lps.embedding_grad(ids, grad, 300), lps.mx4_quantize(grad)
        torch.cuda.synchronize()
        assert torch.equal(a, ea) and torch.equal(b, eb) and torch.equal(c.codes, ec.codes) and torch.equal(c.scales, ec.scales)


def test_refusals(dev):
    x = torch.zeros((4, 64), device=dev)
    t = lps.mx4_quantize(x)
    ids = torch.zeros((3,), dtype=torch.int64, device=dev)
    with pytest.raises(TypeError):
        lps.mx4_quantize(x.double())
    with pytest.raises(ValueError):
        lps.mx4_quantize(x[:, :0])
    with pytest.raises(TypeError):
        lps.mx4_dequantize(t, torch.float64)
    with pytest.raises(ValueError):
        lps.mx4_dequantize(lps.Mx4Tensor(t.codes, t.scales, 65))
    with pytest.raises(TypeError):
        lps.embedding(ids.float(), x)
    with pytest.raises(TypeError):
        lps.embedding(ids, x.double())
    with pytest.raises(ValueError):
        lps.embedding(ids, x[0])
    with pytest.raises(RuntimeError, match="ROCm device"):
        lps.embedding(ids, x.cpu())
    with pytest.raises(ValueError):
        lps.embedding_grad(ids, x, 4)                       # 3 ids, 4 rows
    with pytest.raises(ValueError):
        lps.embedding_grad(ids, x[:3], 0)
    with pytest.raises(ValueError):
        lps.embedding_grad(ids, x[:3], 4, out=x[:, :63])
    with pytest.raises(ValueError):
        lps.embedding_grad(ids, x[:3], 64, out=torch.zeros((64, 64), device=dev).t())
    with pytest.raises(TypeError):
        lps.embedding_grad(ids, x[:3], 4, out=x, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        lps.embedding_grad(ids, x[:3], 4, out=x.clone().requires_grad_())


@pytest.mark.parametrize("n,vocab,hidden,dtype", [(0, 9001, 1023, torch.float32), (3, 70000, 131, torch.float32),
                                                  (900, 30001, 601, torch.bfloat16), (1025, 40000, 517, torch.float16),
                                                  (1500, 1 << 20, 4104, torch.float32), (2, 1 << 20, 4104, torch.float32)])
def test_gradient_writes_every_zero(dev, n, vocab, hidden, dtype):
    """Outputs past the L2s, two of them past 16 GB: rows without a token are zeros
    whatever the memory held, the last id's row is its gradient."""
    torch.full((vocab, hidden), 3.0, dtype=dtype, device=dev)       # freed at once: the same memory
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[n // 2:] = vocab - 1
    grad = torch.ones((n, hidden), dtype=dtype)
    got = lps.embedding_grad(ids.to(dev), grad.to(dev), vocab)
    times = torch.bincount(ids, minlength=vocab)
    assert bool((got[times.nonzero()[:, 0].to(dev)].cpu() == times[times > 0, None]).all())
    got[times.nonzero()[:, 0].to(dev)] = 0
    assert int(torch.count_nonzero(got)) == 0


@pytest.mark.parametrize("n", [3, 1500])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_into_rows_of_a_wider_buffer(dev, n, dtype):
    """The C entry point's new gradient with a row stride: zeros in its rows, nothing beside them."""
    import ctypes
    from lps import _lib
    lib, vocab, hidden = _lib.load(), 9000, 1051
    buf = torch.full((vocab, 1061), 7.0, dtype=dtype, device=dev)
    ids = torch.arange(n, device=dev) % 5
    grad = torch.ones((n, hidden), dtype=dtype, device=dev)
    bytes_ = lib.lps_embedding_grad_workspace_bytes(n, vocab, hidden)
    ws = torch.empty((max(bytes_, 16),), dtype=torch.uint8, device=dev)
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    a = _lib.EmbeddingGradArgs(ids.data_ptr(), grad.data_ptr(), buf[:, 3:].data_ptr(), 8, code, code, n, vocab, hidden,
                               hidden, 1061, 1.0, 0, ws.data_ptr(), bytes_)
    assert lib.lps_embedding_grad(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    times = torch.bincount(ids, minlength=5).to(dtype)
    assert bool((buf[:5, 3:3 + hidden] == times[:, None]).all())
    assert int(torch.count_nonzero(buf[5:, 3:3 + hidden])) == 0
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + hidden:] == 7).all())


@pytest.mark.parametrize("vocab,hidden,dtype", [(4096 * 1024 + 1, 1, torch.bfloat16), (5000001, 3, torch.float32),
                                                (4096 * 1024, 7, torch.float16), (1, 1, torch.float32)])
def test_gradient_of_no_positions(dev, vocab, hidden, dtype):
    """A new gradient of an empty batch is zeros, whatever the vocabulary and the memory held."""
    torch.full((vocab, hidden), 3.0, dtype=dtype, device=dev)       # freed at once: the same memory
    none = torch.empty((0,), dtype=torch.int64, device=dev)
    got = lps.embedding_grad(none, torch.empty((0, hidden), dtype=dtype, device=dev), vocab)
    assert got.shape == (vocab, hidden) and int(torch.count_nonzero(got)) == 0


def test_rows_past_a_grid(dev):
    """More rows than the threads of one launch can take, 16 to a row: every one is
    there (values that their block's scale leaves exact)."""
    rows = (1 << 28) + 5
    x = torch.tensor([1.0, 1.5, -2.0, 3.0, -0.75, 0.0, 48.0], dtype=torch.bfloat16, device=dev)
    ids = torch.arange(rows, dtype=torch.int32, device=dev).remainder_(7)
    all_rows = torch.empty((rows, 1), dtype=torch.bfloat16, device=dev)
    for i in range(0, rows, 1 << 24):
        all_rows[i:i + (1 << 24), 0] = x[ids[i:i + (1 << 24)].long()]
    assert torch.equal(lps.embedding(ids, x[:, None]), all_rows)
    t = lps.mx4_quantize(all_rows)
    assert torch.equal(lps.mx4_dequantize(t), all_rows)


def test_gradient_of_a_huge_vocabulary(dev):
    """The sort's and the zeros' workgroups together at their most: 34 GB of zeros but
    for the ids' rows."""
    vocab, hidden, n = (1 << 30) + 1, 8, 900
    g = torch.Generator().manual_seed(21)
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[:3] = torch.tensor([0, vocab - 1, vocab - 1])
    torch.full((vocab, hidden), 3.0, device=dev)                    # freed at once: the same memory
    got = lps.embedding_grad(ids.to(dev), torch.ones((n, hidden), device=dev), vocab)
    rows, times = ids.unique(return_counts=True)
    assert bool((got[rows.to(dev)].cpu() == times[:, None]).all())
    got[rows.to(dev)] = 0
    for i in range(0, vocab, 1 << 27):
        assert int(torch.count_nonzero(got[i:i + (1 << 27)])) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_tangent(dev, dtype):
    """Forward mode: the tangent's lookup, of a table that requires a gradient and of one that does not."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(14)
    ids = torch.randint(-1, 13, (3, 7), generator=g).to(dev)
    w, t = torch.randn((12, 40), generator=g).to(dev, dtype), torch.randn((12, 40), generator=g).to(dev, dtype)
    with forward_ad.dual_level():
        for table in (w, w.clone().requires_grad_()):
            out = forward_ad.unpack_dual(lps.embedding(ids, forward_ad.make_dual(table, t), scale=1.5))
            assert torch.equal(out.primal, lps.embedding(ids, w, scale=1.5))
            assert torch.equal(out.tangent, lps.embedding(ids, t, scale=1.5))


def test_gradient_out_beside_its_inputs(dev):
    """out and grad in one buffer: refused where they overlap, right where their rows alternate."""
    g = torch.Generator().manual_seed(15)
    ids = torch.randint(0, 30, (30,), generator=g)
    both = torch.randn((30, 40), generator=g)
    buf = both.to(dev)
    with pytest.raises(ValueError, match="overlap"):
        lps.embedding_grad(ids.to(dev), buf[:, 8:28], 30, out=buf[:, 20:])
    before = buf._version
    lps.embedding_grad(ids.to(dev), buf[:, :20], 30, out=buf[:, 20:])
    want, bound = R.gradient(ids, both[:, :20], 30, 1.0, both[:, 20:], torch.float32)
    assert buf._version > before and torch.equal(buf[:, :20].cpu(), both[:, :20])
    assert bool(((buf[:, 20:].double().cpu() - want).abs() <= bound).all())
