"""The vocabulary table's operators on the GPU.

A decode loop uses one table ``[V, H]`` at both of its ends: the sampled
token's row goes in, and the hidden state's products with every row come out
(the reference's ``lm_head``, ``models/qwen3/custom_builder.py:415``).
``embedding`` looks rows up, ``embedding_grad`` is its gradient, and
``mx4_quantize`` gives the table's form in microscaled 4-bit floats (17/64 of
its bf16 bytes), which ``embedding`` and ``lm_head`` take in the table's
place."""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch.autograd import forward_ad

from . import _device as D
from . import _lib

_pack_mx4 = _lib.packer(_lib.Mx4Args)
_pack_embedding = _lib.packer(_lib.EmbeddingArgs)
_pack_grad = _lib.packer(_lib.EmbeddingGradArgs)


class Mx4Tensor(NamedTuple):
    """Rows of microscaled 4-bit floats: ``codes`` uint8 ``[..., 16 * blocks]``
    (element 2 j of a block in the low half of its byte j), ``scales`` uint8
    ``[..., blocks]`` (2^(byte - 127); 255 stands for NaN), blocks of 32 values,
    the last one of a row of ``hidden`` values partly filled (its other codes
    zero)."""

    codes: torch.Tensor
    scales: torch.Tensor
    hidden: int

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.hidden))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def check(self, name: str) -> None:
        """Raises unless the parts are a 4-bit tensor on the GPU."""
        c, s, n = self.codes, self.scales, (self.hidden + 31) // 32
        _on_gpu(c, name + ".codes")
        _on_gpu(s, name + ".scales")
        if c.dtype is not torch.uint8 or s.dtype is not torch.uint8:
            raise TypeError(f"{name}: codes and scales must be uint8")
        cs, ss = c.shape, s.shape
        if n < 1 or len(cs) < 1 or len(ss) != len(cs) or cs[-1] != 16 * n or ss[-1] != n or cs[:-1] != ss[:-1]:
            raise ValueError(f"{name}: codes [..., {16 * n}] and scales [..., {n}] expected for rows of {self.hidden}; "
                             f"got {tuple(cs)}, {tuple(ss)}")
        _same_device(c, s, f"{name}: codes and scales")

    def rows(self):
        """(codes [R, 16 * blocks], scales [R, blocks]) with elements side by
        side and code rows on 16-byte lines."""
        c, s, hidden = self
        if c.dim() != 2:
            c, s = c.reshape(-1, c.shape[-1]), s.reshape(-1, s.shape[-1])
        many, n = c.shape[0] > 1, c.shape[1]
        r, e = c.stride()
        if e != 1 or (many and (r % 16 or r < n)) or c.data_ptr() % 16:
            c = c.clone(memory_format=torch.contiguous_format)
        r, e = s.stride()
        if (e != 1 and n > 16) or (many and r < n // 16):
            s = s.contiguous()
        return c, s


def _on_gpu(t: torch.Tensor, name: str) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        D.require_device(t, name)


def _flat_rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, H] with a row's elements side by side and rows apart (a
    broadcast gradient's are not)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    r, e = x.stride()
    n, h = x.shape
    if (e != 1 and h > 1) or (r < h and n > 1):
        x = x.contiguous()
    return x


def _same_device(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    if a.get_device() != b.get_device():
        raise ValueError(f"{what} are on different devices: {a.device}, {b.device}")


def _has_tangent(t: torch.Tensor) -> bool:
    """Whether t carries a forward-mode derivative (it can where a level of them is open)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _no_derivative(t: torch.Tensor, name: str, call: str) -> None:
    """Raises where t asks for a derivative: the call has none, and would lose it."""
    if (t.requires_grad and torch.is_grad_enabled()) or _has_tangent(t):
        raise ValueError(f"{call} has no derivative in {name}, which requires a gradient or carries a tangent; "
                         "detach it, or call without gradients")


def _share_memory(a, b) -> bool:
    """Whether two sets of rows, each (address, rows, bytes from row to row, bytes of
    one), have a byte in common.  Rows of one set do not overlap each other."""
    if a[1] > b[1]:
        a, b = b, a
    (p, n, s, k), (q, m, t, j) = a, b
    if n == 0 or p + (n - 1) * s + k <= q or q + (m - 1) * t + j <= p:
        return False
    # of each row of the smaller set: the last row of the other that begins before its end
    x = p - q + s * torch.arange(n, dtype=torch.int64, device="cpu")
    last = torch.div(x + (k - 1), max(t, 1), rounding_mode="floor").clamp_(max=m - 1)
    return bool(((last >= 0) & (last * t + j > x)).any())


def _call(name: str, args: bytes, device: torch.device) -> None:
    """The entry point on the device's current stream; raises for its return code."""
    fn = getattr(_lib.load(), name)
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with D.guard(device):
            rc = fn(args, D.stream_of(device))
    if rc:
        _lib.check(rc, name)


def _sizes(*n: int) -> None:
    """The C ABI counts in 32 bits."""
    if max(n) > 0x7FFFFFFF:
        raise ValueError(f"sizes of at most {0x7FFFFFFF} expected; got {max(n)}")


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """``x [..., H]`` (float32, bfloat16 or float16) to microscaled 4-bit floats
    along its last dimension.

    A block of 32 values has the scale 2^s, s = max(floor(log2(largest
    magnitude)) - 2, -126), and the codes of the nearest of 0, 0.5, 1, 1.5, 2, 3,
    4, 6 to ``|x| / 2^s`` (ties to the even code, 6 above it; signs are kept).  A
    block with a value that is not finite becomes NaN.  ``H`` need not be a
    multiple of 32.  Codes and scales are whole numbers: they carry no gradient of
    ``x``."""
    _on_gpu(x, "x")
    code = D.code_of(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x [..., H] with H >= 1 expected; got {tuple(x.shape)}")
    xf = _flat_rows(x)
    device = x.device
    rows, hidden = xf.shape
    _sizes(rows, hidden)
    n = (hidden + 31) // 32
    codes = torch.empty((rows, 16 * n), dtype=torch.uint8, device=device)
    # scale rows on 4-byte lines: the LM head reads four at a time
    scales = torch.empty((rows, n + -n % 4), dtype=torch.uint8, device=device)
    if n % 4:
        scales = scales[:, :n]
    if rows:
        _call("lps_mx4_quantize",
              _pack_mx4(xf.data_ptr(), codes.data_ptr(), scales.data_ptr(), code, rows, hidden,
                        xf.stride(0) if rows > 1 else hidden, 16 * n, n + -n % 4), device)
    if xf is not x:
        lead = x.shape[:-1]
        if len(lead) != 1:
            codes, scales = codes.view(*lead, 16 * n), scales.unflatten(0, lead) if lead else scales[0]
    return Mx4Tensor(codes, scales, hidden)


def mx4_dequantize(t: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values ``[..., H]`` of a 4-bit tensor, in ``dtype`` (every one that
    ``mx4_quantize`` gives is exact in bfloat16 and float32; those past float32's
    range, which scale bytes 253 and 254 can hold, are infinities)."""
    t.check("t")
    code = D.code_of(dtype)
    codes, scales = t.rows()
    rows, device, hidden = codes.shape[0], codes.device, t.hidden
    _sizes(rows, hidden)
    out = torch.empty((rows, hidden), dtype=dtype, device=device)
    if rows:
        many = rows > 1
        _call("lps_mx4_dequantize",
              _pack_mx4(out.data_ptr(), codes.data_ptr(), scales.data_ptr(), code, rows, hidden, hidden,
                        codes.stride(0) if many else codes.shape[1], scales.stride(0) if many else scales.shape[1]), device)
    return out if t.codes.dim() == 2 else out.reshape(t.shape)


def _ids(ids: torch.Tensor) -> torch.Tensor:
    """ids as a vector of neighbouring elements."""
    _on_gpu(ids, "ids")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"ids must be int64 or int32; got {ids.dtype}")
    return ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()


def _embedding(ids: torch.Tensor, table: Union[torch.Tensor, Mx4Tensor], scale: float,
               out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    flat = _ids(ids)
    if isinstance(table, Mx4Tensor):
        table.check("table")
        if table.codes.dim() != 2:
            raise ValueError(f"table [V, H] expected; got {tuple(table.shape)}")
        rows, scales = table.rows()
        hidden, code, dtype = table.hidden, _lib.LPS_DTYPE_MX4, out_dtype or torch.bfloat16
        vocab = rows.shape[0]
        sp, ss = scales.data_ptr(), scales.stride(0) if vocab > 1 else scales.shape[1]
    else:
        _on_gpu(table, "table")
        code, dtype = D.code_of(table.dtype), out_dtype or table.dtype
        if table.dim() != 2 or table.shape[1] < 1:
            raise ValueError(f"table [V, H] expected; got {tuple(table.shape)}")
        rows = _flat_rows(table)
        vocab, hidden = rows.shape
        sp = ss = 0
    _same_device(ids, rows, "ids and table")
    if vocab < 1:
        raise ValueError("the table has no rows")
    device, n = rows.device, flat.shape[0]
    _sizes(n, vocab, hidden)
    out_code = D.code_of(dtype)
    out = torch.empty((n, hidden), device=device, dtype=dtype)
    if n:
        _call("lps_embedding",
              _pack_embedding(flat.data_ptr(), rows.data_ptr(), sp, out.data_ptr(), flat.element_size(), code, out_code, n,
                              vocab, hidden, rows.stride(0) if vocab > 1 else rows.shape[1], ss, hidden, scale), device)
    return out if flat is ids else out.reshape(*ids.shape, hidden)


class _Embedding(torch.autograd.Function):
    """The lookup with its derivatives in the table: it is linear in it."""

    @staticmethod
    def forward(ctx, ids, table, scale, out_dtype):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.vocab, ctx.scale, ctx.dtype, ctx.out_dtype = table.shape[0], scale, table.dtype, out_dtype
        return _embedding(ids, table, scale, out_dtype)

    @staticmethod
    def jvp(ctx, _, tangent, *__):
        (ids,) = ctx.saved_tensors
        return embedding(ids, tangent, ctx.scale, ctx.out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return None, embedding_grad(ids, grad, ctx.vocab, scale=ctx.scale, dtype=ctx.dtype), None, None


def embedding(ids: torch.Tensor, table: Union[torch.Tensor, Mx4Tensor], scale: float = 1.0,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale * table[ids]``: ``[..., H]`` for ``ids [...]`` (int64 or int32) and
    a table ``[V, H]`` in float32, bfloat16, float16 or 4 bits; fp32 arithmetic,
    rounded once to ``out_dtype`` (default: the table's type, bfloat16 for 4
    bits).  Ids outside ``[0, V)``, -1 among them, give zeros.  A table that
    requires a gradient gets it from ``embedding_grad``; the forward-mode
    derivative of one that carries a tangent is the tangent's lookup."""
    if isinstance(table, torch.Tensor) and ((table.requires_grad and torch.is_grad_enabled()) or _has_tangent(table)):
        return _Embedding.apply(ids, table, scale, out_dtype)
    return _embedding(ids, table, scale, out_dtype)


def embedding_grad(ids: torch.Tensor, grad: torch.Tensor, vocab: int, scale: float = 1.0,
                   dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``embedding`` in its table: row v is ``scale`` times the sum
    of ``grad [..., H]`` over the positions of ``ids [...]`` that hold v (ids
    outside ``[0, vocab)`` add nothing), summed in fp32 and rounded once.

    A new tensor ``[vocab, H]`` of ``dtype`` (default: ``grad``'s), or, with
    ``out``, added to ``out [vocab, H]`` (of which the rows without a position are
    left alone) and ``out`` returned (it shares no memory with ``grad`` and
    ``ids``).  The order of the sum depends on ids and
    sizes alone: equal calls give equal bits.  It has no derivative itself: a
    ``grad`` or ``out`` that asks for one is refused."""
    flat = _ids(ids)
    _on_gpu(grad, "grad")
    code = D.code_of(grad.dtype)
    _no_derivative(grad, "grad", "embedding_grad")
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape or grad.shape[-1] < 1:
        raise ValueError(f"ids [...] and grad [..., H] expected; got {tuple(ids.shape)}, {tuple(grad.shape)}")
    if vocab < 1:
        raise ValueError(f"vocab must be at least 1; got {vocab}")
    _same_device(ids, grad, "ids and grad")
    device, hidden, n = grad.device, grad.shape[-1], flat.shape[0]
    _sizes(n, vocab, hidden)
    g = _flat_rows(grad)
    if out is None:
        dtype = dtype or grad.dtype
        out_code = D.code_of(dtype)
        res = torch.empty((vocab, hidden), dtype=dtype, device=device)
    else:
        _on_gpu(out, "out")
        _same_device(out, grad, "out and grad")
        if dtype is not None and dtype != out.dtype:
            raise TypeError(f"dtype {dtype} and out of {out.dtype}")
        out_code = D.code_of(out.dtype)
        if out.shape != (vocab, hidden) or (hidden > 1 and out.stride(1) != 1) or (vocab > 1 and out.stride(0) < hidden):
            raise ValueError(f"out [{vocab}, {hidden}] with rows of neighbouring elements expected; got "
                             f"{tuple(out.shape)}, strides {out.stride()}")
        _no_derivative(out, "out", "embedding_grad")
        res = out
    gs, rs = g.stride(0) if n > 1 else hidden, res.stride(0) if vocab > 1 else hidden
    if out is not None:
        rows = (res.data_ptr(), vocab, rs * res.element_size(), hidden * res.element_size())
        if (_share_memory((g.data_ptr(), n, gs * g.element_size(), hidden * g.element_size()), rows)
                or _share_memory((flat.data_ptr(), 1 if n else 0, 0, n * flat.element_size()), rows)):
            raise ValueError("out overlaps grad or ids in memory")
    need = _lib.load().lps_embedding_grad_workspace_bytes(n, vocab, hidden)
    ws = torch.empty((need,), dtype=torch.uint8, device=device) if need else None
    _call("lps_embedding_grad",
          _pack_grad(flat.data_ptr(), g.data_ptr(), res.data_ptr(), flat.element_size(), code, out_code, n, vocab, hidden,
                     gs, rs, scale, 0 if out is None else 1, D.ptr(ws), need), device)
    if out is not None:
        torch.autograd.graph.increment_version(out)   # written behind autograd's back
    return res
