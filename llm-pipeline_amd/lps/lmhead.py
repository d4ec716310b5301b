"""The LM-head projection with the softmax-statistics epilogue on the GPU.

The reference's logits producer is ``self.lm_head(hidden_states)``
(``models/qwen3/custom_builder.py:415``, ``models/qwen3_5/model.py:263``), an
``nn.Linear`` without bias.  ``lm_head`` computes the same projection with the
``lps_lm_head`` MFMA kernel and, while the tile is in registers, each row's
``(max, sum(exp(v - max)))`` over every block of 128 vocabulary columns, so a
softmax of the logits (``fused_softmax(logits, row_stats=stats)``) needs one
streaming pass instead of a statistics pass first."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _device as D
from . import _lib
from .vocab_table import Mx4Tensor, _call, _no_derivative, _on_gpu, _same_device, _sizes

_pack_mx4 = _lib.packer(_lib.LmHeadMx4Args)


def lm_head(hidden: Union[torch.Tensor, Mx4Tensor], weight: Union[torch.Tensor, Mx4Tensor], out_dtype: Optional[torch.dtype] = None,
            return_stats: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``hidden [..., H] @ weight[V, H].T`` -> logits ``[..., V]`` (fp32
    accumulation, stored in ``out_dtype``, default the input dtype).  Inputs:
    bf16 or fp16, the same dtype, ``H`` a multiple of 16.  ``return_stats``
    also returns ``[..., ceil(V / 128), 2]`` float32 block statistics
    ``(max, sum(exp(v - max)))`` of the stored logits.  The logits carry no
    gradient.

    ``weight`` may be 4-bit (``mx4_quantize``): then ``H`` is any number,
    ``hidden`` bf16, fp16 or 4-bit itself, and ``out_dtype`` bfloat16 by default
    for 4-bit ``hidden``.  The products are exact and summed in fp32 (to a
    16-bit ``hidden`` a weight past float32's range is an infinity).  A 16-bit
    ``hidden`` that asks for a derivative is refused."""
    if isinstance(weight, Mx4Tensor) or isinstance(hidden, Mx4Tensor):
        return _lm_head_mx4(hidden, weight, out_dtype, return_stats)
    D.require_device(hidden, "hidden")
    D.require_device(weight, "weight")
    if weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden [..., H] and weight [V, H] expected; got {tuple(hidden.shape)}, {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("hidden and weight must both be bfloat16 or both float16")
    V, H = weight.shape
    lead = hidden.shape[:-1]
    x = hidden.reshape(-1, H)
    if x.stride(-1) != 1 or (x.shape[0] > 1 and x.stride(0) % 8) or x.data_ptr() % 16:
        x = x.contiguous()
    w = weight
    if w.stride(-1) != 1 or w.stride(0) % 8 or w.data_ptr() % 16:
        w = w.contiguous()
    M = x.shape[0]
    od = out_dtype or hidden.dtype
    out = torch.empty((M, V), dtype=od, device=hidden.device)
    G = (V + _lib.LMHEAD_BLOCK_COLS - 1) // _lib.LMHEAD_BLOCK_COLS
    stats = torch.empty((M, G, 2), dtype=torch.float32, device=hidden.device) if return_stats else None
    a = _lib.LmHeadArgs()
    a.x, a.w, a.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
    a.stats = D.ptr(stats)
    a.dtype = D.dtype_code(x)
    a.out_dtype = D.dtype_code(out)
    a.rows, a.vocab, a.hidden = M, V, H
    a.x_stride = x.stride(0) if M > 1 else H
    a.w_stride = w.stride(0)
    a.out_stride = V
    if M:
        with D.guard(hidden.device):
            rc = _lib.load().lps_lm_head(ctypes.byref(a), D.stream_of(hidden.device))
        _lib.check(rc, "lps_lm_head")
    out = out.reshape(*lead, V)
    if return_stats:
        return out, stats.reshape(*lead, G, 2)
    return out


_MX4_MAX_STRIDE = 1 << 23   # bytes between rows (include/lps.h)


def _words(s: torch.Tensor) -> torch.Tensor:
    """Scales with rows on 4-byte lines, as the kernel reads them."""
    rows, n = s.shape
    r = s.stride(0) if rows > 1 else 0
    if s.data_ptr() % 4 == 0 and r % 4 == 0 and r <= _MX4_MAX_STRIDE:
        return s
    out = torch.empty((rows, n + -n % 4), dtype=torch.uint8, device=s.device)[:, :n]
    return out.copy_(s)


def _lm_head_mx4(hidden, weight, out_dtype, return_stats):
    if not isinstance(weight, Mx4Tensor):
        raise TypeError("a 4-bit hidden state needs a 4-bit weight")
    weight.check("weight")
    H = weight.hidden
    if isinstance(hidden, Mx4Tensor):
        hidden.check("hidden")
        code, od = _lib.LPS_DTYPE_MX4, out_dtype or torch.bfloat16
        lead, width = hidden.codes.shape[:-1], hidden.hidden
        x, xs = hidden.rows()
        xs = _words(xs)
        xp, xss = xs.data_ptr(), xs.stride(0)
    else:
        _on_gpu(hidden, "hidden")
        if hidden.dtype is not torch.bfloat16 and hidden.dtype is not torch.float16:
            raise TypeError("hidden must be bfloat16, float16 or an Mx4Tensor")
        _no_derivative(hidden, "hidden", "lm_head over a 4-bit weight")
        code, od = D.code_of(hidden.dtype), out_dtype or hidden.dtype
        lead, width = hidden.shape[:-1], hidden.shape[-1] if hidden.dim() else 0
        x, xp, xss = hidden, 0, 0
        if x.dim() != 2 and width:
            x = x.reshape(-1, width)
    if width != H or weight.codes.dim() != 2 or weight.codes.shape[0] < 1:
        raise ValueError(f"hidden [..., H] and weight [V, H] expected; got {tuple(hidden.shape)}, {tuple(weight.shape)}")
    _same_device(x, weight.codes, "hidden and weight")
    M = x.shape[0]
    if code != _lib.LPS_DTYPE_MX4:
        r, e = x.stride()
        # rows on 16-byte lines: a copy that lies so
        if (e != 1 and H > 1) or x.data_ptr() % 16 or (M > 1 and (r % 8 or not H <= r <= max(_MX4_MAX_STRIDE // 2, H + 7))):
            x = torch.empty((M, H + -H % 8), dtype=x.dtype, device=x.device)[:, :H].copy_(x)
    elif M > 1 and x.stride(0) > _MX4_MAX_STRIDE:
        x = x.contiguous()
    w, ws = weight.rows()
    if w.shape[0] > 1 and w.stride(0) > _MX4_MAX_STRIDE:
        w = w.contiguous()
    ws = _words(ws)
    device, V = w.device, w.shape[0]
    _sizes(M, V, H)
    out_code = D.code_of(od)
    out = torch.empty((M, V), dtype=od, device=device)
    G = (V + _lib.LMHEAD_BLOCK_COLS - 1) // _lib.LMHEAD_BLOCK_COLS
    stats = torch.empty((M, G, 2), dtype=torch.float32, device=device) if return_stats else None
    # (16-bit rows of more than 8 MiB: one to a call)
    step = M if code == _lib.LPS_DTYPE_MX4 or M < 2 or x.stride(0) <= _MX4_MAX_STRIDE // 2 else 1
    for m in range(0, M, step or 1):
        if m:
            xm, op, sp = x[m:].data_ptr(), out[m:].data_ptr(), D.ptr(None if stats is None else stats[m:])
        else:
            xm, op, sp = x.data_ptr(), out.data_ptr(), D.ptr(stats)
        _call("lps_lm_head_mx4",
              _pack_mx4(xm, xp, w.data_ptr(), ws.data_ptr(), op, sp, code, out_code, step, V, H,
                        x.stride(0), xss, w.stride(0), ws.stride(0), V), device)
    if len(lead) != 1:
        out = out.reshape(*lead, V)
        stats = None if stats is None else stats.reshape(*lead, G, 2)
    return (out, stats) if return_stats else out
