"""The vocabulary table's operators from their definitions, in 64 bits on the
CPU: what the kernels' tests compare with."""

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# half a step of a type's rounding, relative to the value, and half its smallest step
HALF = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
        torch.float16: (2.0 ** -11, 2.0 ** -25)}


def power(s):
    return torch.ldexp(torch.ones((), dtype=torch.float64), s)


def hard_values(rows, hidden, dtype, g):
    """Values at every border of the 4-bit form: magnitudes over the whole range
    of exponents, ties, zeros of both signs, subnormals, blocks with infinities
    and NaN."""
    x = torch.randn((rows, hidden), generator=g, dtype=torch.float64)
    x *= 2.0 ** torch.randint(-30, 12, (rows, 1), generator=g).double()
    tie = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 6.0, 7.0, 0.0], dtype=torch.float64)
    pick = torch.randint(0, 11, (rows, hidden), generator=g)
    sign = torch.where(torch.rand((rows, hidden), generator=g) < 0.5, -1.0, 1.0).double()
    x[0] = (tie[pick] * sign)[0]
    if rows > 2:
        x[2] *= 2.0 ** -100 if dtype != torch.float16 else 2.0 ** -12
        x[2, ::3] = -0.0
    if rows > 3:
        x[3] = 0.0
    out = x.to(dtype)
    if rows > 4:
        out[4, hidden // 2] = float("nan")
        out[4, 0] = float("inf")
    if rows > 5:
        out[5, hidden - 1] = float("-inf")
    return out


def quantise(x):
    """(codes [R, 16 blocks], scales [R, blocks]) of x [R, H]."""
    rows, hidden = x.shape
    nb = -(-hidden // 32)
    d = torch.zeros((rows, nb * 32), dtype=torch.float64)
    d[:, :hidden] = x.double()
    d = d.reshape(rows, nb, 32)
    top = d.abs().amax(2)
    fine = torch.isfinite(top)
    s = (torch.frexp(torch.where(fine, top, 0.0)).exponent - 3).clamp(min=-126)
    s = torch.where(top == 0, -126, s)
    a = d.abs() / power(s).unsqueeze(2)
    code = torch.zeros(d.shape, dtype=torch.uint8)
    for c in range(1, 8):   # past the middle to the lower code, or on it when c is even
        mid = (VALUES[c - 1] + VALUES[c]) / 2
        code += (a > mid) | ((a == mid) & (c % 2 == 0))
    code += 8 * torch.signbit(d).to(torch.uint8)
    code *= fine.unsqueeze(2)
    code = code.reshape(rows, nb * 16, 2)
    return code[:, :, 0] | (code[:, :, 1] << 4), torch.where(fine, s + 127, 255).to(torch.uint8)


def values(codes, scales, hidden):
    """The values [R, H] that codes and scales stand for."""
    c = torch.stack((codes & 15, codes >> 4), 2).reshape(*scales.shape, 32).long()
    v = torch.where(c >= 8, -1.0, 1.0) * VALUES[c & 7]
    s = torch.where(scales == 255, float("nan"), power(scales.int() - 127))
    return (v * s.unsqueeze(2)).flatten(1)[:, :hidden]


def gradient(ids, grad, vocab, scale, out, out_dtype):
    """(out + scale * sums of grad by id, how far a result may be off): the fp32
    sums of k terms by (k - 1) 2^-24 of the sum of magnitudes, the product with
    the scale, the sum with out and the store by half a step each."""
    at = torch.nonzero((ids >= 0) & (ids < vocab)).reshape(-1)
    i = ids[at].long()
    want = torch.zeros((vocab, grad.shape[1]), dtype=torch.float64).index_add_(0, i, grad[at].double() * scale)
    mag = torch.zeros((vocab, grad.shape[1]), dtype=torch.float64).index_add_(0, i, grad[at].double().abs() * abs(scale))
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, i, torch.ones(len(at), dtype=torch.float64))
    if out is not None:
        want = want + out.double()
    rel, least = HALF[out_dtype]
    bound = (count.unsqueeze(1) + 2) * 2.0 ** -24 * mag + want.abs() * (rel + 2.0 ** -23) * 1.01 + least
    return want, bound


def extreme_scales(V, H, M, dtype):
    """(codes, scales, x) of a head whose weights' scales are the largest and the
    smallest, one value a row: products of one term each, no sum to round."""
    nb = -(-H // 32)
    codes = torch.zeros((V, 16 * nb), dtype=torch.uint8)
    scales = torch.full((V, nb), 127, dtype=torch.uint8)
    n = torch.arange(V)
    at = (n * 37) % H                                      # the row's column
    code = (1 + n % 7 + 8 * (n // 7 % 2)).to(torch.uint8)
    codes[n, at // 2] = code << (4 * (at % 2)).to(torch.uint8)
    scales[n, at // 32] = torch.tensor([254, 253, 252, 0, 1, 2, 60, 141, 103])[n % 9].to(torch.uint8)
    # 8 bits, 11 bits, the largest, the smallest (fp16's), powers of two
    v = torch.tensor([1.0, -1.25, 1.0 + 2.0 ** -7, 3.0 if dtype == torch.bfloat16 else 1.0 + 2.0 ** -10, 2.0 ** 15, -2.0 ** -24,
                      2.0 ** -3])
    x = v[(torch.arange(M)[:, None] + torch.arange(H)) % 7].to(dtype)
    x[0, 37], x[M - 1, H - 1] = float("inf"), float("-inf")
    return codes, scales, x


def extreme_products(codes, scales, x):
    """x times those weights as fp32: a weight past its range is an infinity."""
    w = values(codes, scales, x.shape[1]).float().double()
    n = torch.arange(w.shape[0])
    at = (n * 37) % x.shape[1]
    out = x.double()[:, at] * w[n, at]
    # (an infinite state times one of the row's zeros)
    infinite = torch.isinf(x.double())
    return torch.where(infinite.sum(1, keepdim=True) > infinite[:, at].long(), float("nan"), out).float().double()


def check_extreme(out, ref):
    """Equal but for products under fp32's normal range, which matrix cores need not keep."""
    out, fine = out.double().cpu(), torch.isfinite(ref)
    assert torch.equal(out[~fine].nan_to_num(nan=0.125), ref[~fine].nan_to_num(nan=0.125))
    assert bool(((out - ref)[fine].abs() <= torch.where(ref[fine].abs() < 2.0 ** -126, 2.0 ** -126, 0.0)).all())
