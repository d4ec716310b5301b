"""The vocabulary table's operators on the GPU.

A decode loop uses one table ``[V, H]`` at both of its ends: the sampled
token's row goes in (the reference's ``nn.Embedding``,
``models/qwen3/custom_builder.py``) and the hidden state's products with every
row come out (``lm_head``, the same file ``:415``).  ``embedding`` looks rows
up, ``embedding_grad`` is its gradient, and ``mx4_quantize`` gives the table's
form in microscaled 4-bit floats (17/64 of its bf16 bytes), which
``embedding`` and ``lm_head`` take in the table's place."""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Union

import torch

from . import _device as D
from . import _lib


def _blocks(hidden: int) -> int:
    return -(-hidden // _lib.LPS_MX4_BLOCK)


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
        D.require_device(self.codes, name + ".codes")
        D.require_device(self.scales, name + ".scales")
        if self.codes.dtype != torch.uint8 or self.scales.dtype != torch.uint8:
            raise TypeError(f"{name}: codes and scales must be uint8")
        n = _blocks(self.hidden)
        if self.hidden < 1 or self.codes.dim() < 1 or self.codes.shape[-1] != 16 * n \
                or self.scales.shape != (*self.codes.shape[:-1], n):
            raise ValueError(f"{name}: codes [..., {16 * n}] and scales [..., {n}] expected for rows of {self.hidden}; "
                             f"got {tuple(self.codes.shape)}, {tuple(self.scales.shape)}")
        if self.codes.device != self.scales.device:
            raise ValueError(f"{name}: codes and scales are on different devices")

    def rows(self):
        """(codes [R, 16 * blocks], scales [R, blocks]) with elements side by
        side and code rows on 16-byte lines."""
        c, s = self.codes, self.scales
        if c.dim() != 2:
            c, s = c.reshape(-1, c.shape[-1]), s.reshape(-1, s.shape[-1])
        if c.stride(1) != 1 or (c.shape[0] > 1 and (c.stride(0) % 16 or c.stride(0) < c.shape[1])) or c.data_ptr() % 16:
            c = c.clone(memory_format=torch.contiguous_format)
        if (s.stride(1) != 1 and s.shape[1] > 1) or (s.shape[0] > 1 and s.stride(0) < s.shape[1]):
            s = s.contiguous()
        return c, s


def _flat_rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, H] with a row's elements side by side and rows apart (a
    broadcast gradient's are not)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if (x.stride(1) != 1 and x.shape[1] > 1) or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def _same_device(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    if a.device != b.device:
        raise ValueError(f"{what} are on different devices: {a.device}, {b.device}")


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """``x [..., H]`` (float32, bfloat16 or float16) to microscaled 4-bit floats
    along its last dimension.

    A block of 32 values has the scale 2^s, s = max(floor(log2(largest
    magnitude)) - 2, -126), and the codes of the nearest of 0, 0.5, 1, 1.5, 2, 3,
    4, 6 to ``|x| / 2^s`` (ties to the even code, 6 above it; signs are kept).  A
    block with a value that is not finite becomes NaN.  ``H`` need not be a
    multiple of 32."""
    D.require_device(x, "x")
    code = D.dtype_code(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x [..., H] with H >= 1 expected; got {tuple(x.shape)}")
    lead, hidden = x.shape[:-1], x.shape[-1]
    xf = _flat_rows(x)
    n, rows = _blocks(hidden), xf.shape[0]
    codes = torch.empty((rows, 16 * n), dtype=torch.uint8, device=x.device)
    # scale rows on 4-byte lines: the LM head reads four at a time
    scales = torch.empty((rows, n + -n % 4), dtype=torch.uint8, device=x.device)[:, :n]
    if rows:
        a = _lib.Mx4Args(xf.data_ptr(), codes.data_ptr(), scales.data_ptr(), code, rows, hidden,
                         xf.stride(0) if rows > 1 else hidden, codes.stride(0), scales.stride(0))
        with D.guard(x.device):
            rc = _lib.load().lps_mx4_quantize(ctypes.byref(a), D.stream_of(x.device))
        _lib.check(rc, "lps_mx4_quantize")
    if len(lead) != 1:
        codes, scales = codes.view(*lead, 16 * n), scales.unflatten(0, lead) if lead else scales[0]
    return Mx4Tensor(codes, scales, hidden)


def mx4_dequantize(t: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values ``[..., H]`` of a 4-bit tensor, in ``dtype`` (every one is
    exact in bfloat16 and float32)."""
    t.check("t")
    codes, scales = t.rows()
    rows = codes.shape[0]
    out = torch.empty((rows, t.hidden), dtype=dtype, device=codes.device)
    code = D.dtype_code(out)
    if rows:
        a = _lib.Mx4Args(out.data_ptr(), codes.data_ptr(), scales.data_ptr(), code, rows, t.hidden, t.hidden,
                         codes.stride(0) if rows > 1 else codes.shape[1], scales.stride(0) if rows > 1 else scales.shape[1])
        with D.guard(codes.device):
            rc = _lib.load().lps_mx4_dequantize(ctypes.byref(a), D.stream_of(codes.device))
        _lib.check(rc, "lps_mx4_dequantize")
    return out.reshape(t.shape)


def _ids(ids: torch.Tensor) -> torch.Tensor:
    D.require_device(ids, "ids")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32; got {ids.dtype}")
    return ids.reshape(-1).contiguous()


def _embedding(ids: torch.Tensor, table: Union[torch.Tensor, Mx4Tensor], scale: float,
               out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    flat = _ids(ids)
    a = _lib.EmbeddingArgs()
    if isinstance(table, Mx4Tensor):
        table.check("table")
        if table.codes.dim() != 2:
            raise ValueError(f"table [V, H] expected; got {tuple(table.shape)}")
        rows, scales = table.rows()
        hidden = table.hidden
        a.dtype, a.scales = _lib.LPS_DTYPE_MX4, scales.data_ptr()
        a.scales_stride = scales.stride(0) if rows.shape[0] > 1 else scales.shape[1]
    else:
        D.require_device(table, "table")
        if table.dim() != 2 or table.shape[1] < 1:
            raise ValueError(f"table [V, H] expected; got {tuple(table.shape)}")
        a.dtype = D.dtype_code(table)
        rows, hidden = _flat_rows(table), table.shape[1]
    _same_device(ids, rows, "ids and table")
    if rows.shape[0] < 1:
        raise ValueError("the table has no rows")
    out = torch.empty((flat.shape[0], hidden), device=rows.device,
                      dtype=out_dtype or (torch.bfloat16 if isinstance(table, Mx4Tensor) else table.dtype))
    a.out_dtype = D.dtype_code(out)
    if flat.shape[0]:
        a.ids, a.table, a.out = flat.data_ptr(), rows.data_ptr(), out.data_ptr()
        a.id_bytes = flat.element_size()
        a.n, a.vocab, a.hidden = flat.shape[0], rows.shape[0], hidden
        a.table_stride = rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]
        a.out_stride = hidden
        a.scale = scale
        with D.guard(rows.device):
            rc = _lib.load().lps_embedding(ctypes.byref(a), D.stream_of(rows.device))
        _lib.check(rc, "lps_embedding")
    return out.reshape(*ids.shape, hidden)


class _Embedding(torch.autograd.Function):
    """The lookup with its gradient in the table."""

    @staticmethod
    def forward(ctx, ids, table, scale, out_dtype):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale, ctx.dtype = table.shape[0], scale, table.dtype
        return _embedding(ids, table, scale, out_dtype)

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
    requires a gradient gets it from ``embedding_grad``."""
    if isinstance(table, torch.Tensor) and table.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, table, scale, out_dtype)
    return _embedding(ids, table, scale, out_dtype)


def embedding_grad(ids: torch.Tensor, grad: torch.Tensor, vocab: int, scale: float = 1.0,
                   dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``embedding`` in its table: row v is ``scale`` times the sum
    of ``grad [..., H]`` over the positions of ``ids [...]`` that hold v (ids
    outside ``[0, vocab)`` add nothing), summed in fp32 and rounded once.

    A new tensor ``[vocab, H]`` of ``dtype`` (default: ``grad``'s), or, with
    ``out``, added to ``out [vocab, H]`` (of which the rows without a position are
    left alone) and ``out`` returned.  The order of the sum depends on ids and
    sizes alone: equal calls give equal bits."""
    flat = _ids(ids)
    D.require_device(grad, "grad")
    code = D.dtype_code(grad)
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape or grad.shape[-1] < 1:
        raise ValueError(f"ids [...] and grad [..., H] expected; got {tuple(ids.shape)}, {tuple(grad.shape)}")
    if vocab < 1:
        raise ValueError(f"vocab must be at least 1; got {vocab}")
    _same_device(ids, grad, "ids and grad")
    hidden, n = grad.shape[-1], flat.shape[0]
    g = _flat_rows(grad)
    if out is None:
        res = torch.empty((vocab, hidden), dtype=dtype or grad.dtype, device=grad.device)
    else:
        D.require_device(out, "out")
        _same_device(out, grad, "out and grad")
        if dtype is not None and dtype != out.dtype:
            raise TypeError(f"dtype {dtype} and out of {out.dtype}")
        if tuple(out.shape) != (vocab, hidden) or (hidden > 1 and out.stride(1) != 1) or (vocab > 1 and out.stride(0) < hidden):
            raise ValueError(f"out [{vocab}, {hidden}] with rows of neighbouring elements expected; got "
                             f"{tuple(out.shape)}, strides {out.stride()}")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out requires a gradient; pass its .grad, or a detached tensor")
        res = out
    lib = _lib.load()
    need = lib.lps_embedding_grad_workspace_bytes(n, vocab, hidden)
    ws = torch.empty((need,), dtype=torch.uint8, device=grad.device)
    a = _lib.EmbeddingGradArgs()
    a.ids, a.grad, a.out = flat.data_ptr(), g.data_ptr(), res.data_ptr()
    a.id_bytes, a.dtype, a.out_dtype = flat.element_size(), code, D.dtype_code(res)
    a.n, a.vocab, a.hidden = n, vocab, hidden
    a.grad_stride = g.stride(0) if n > 1 else hidden
    a.out_stride = res.stride(0) if vocab > 1 else hidden
    a.scale, a.accumulate = scale, int(out is not None)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    with D.guard(grad.device):
        rc = lib.lps_embedding_grad(ctypes.byref(a), D.stream_of(grad.device))
    _lib.check(rc, "lps_embedding_grad")
    return res
