"""CPU checks of the vocabulary table's C ABI and host layer: struct layouts,
argument errors (reported before any launch) and refusals of CPU tensors."""

import ctypes

import pytest
import torch

from tests.test_abi import _c_layout, lib  # noqa: F401


@pytest.mark.parametrize("cname,pyname", [("lps_mx4_args", "Mx4Args"), ("lps_embedding_args", "EmbeddingArgs"),
                                         ("lps_embedding_grad_args", "EmbeddingGradArgs"),
                                         ("lps_lm_head_mx4_args", "LmHeadMx4Args")])
def test_struct_layout_matches_c(cname, pyname):
    from lps import _lib
    py = getattr(_lib, pyname)
    names = [f[0] for f in py._fields_]
    size, offs = _c_layout(cname, names)
    assert ctypes.sizeof(py) == size
    assert [getattr(py, n).offset for n in names] == offs


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 2), (dict(dtype=-1), 2), (dict(rows=-1), 1), (dict(hidden=0), 1), (dict(hidden=1 << 25), 1),
    (dict(rows=0, x=0), 0), (dict(x=0), 1), (dict(codes=0), 1), (dict(scales=0), 1), (dict(x=0x1001), 1),
    (dict(codes=0x2002), 1), (dict(codes_stride=50), 1), (dict(codes_stride=28), 1), (dict(x_stride=39), 1),
    (dict(scales_stride=1), 1)])
@pytest.mark.parametrize("entry", ["lps_mx4_quantize", "lps_mx4_dequantize"])
def test_mx4_argument_errors(lib, entry, kw, code):  # noqa: F811
    from lps import _lib
    a = _lib.Mx4Args(0x1000, 0x2000, 0x3000, 1, 4, 40, 40, 32, 2)
    for k, v in kw.items():
        setattr(a, k, v)
    assert getattr(lib, entry)(ctypes.byref(a), None) == code
    assert getattr(lib, entry)(None, None) == 1


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=4), 2), (dict(out_dtype=3), 2), (dict(id_bytes=2), 1), (dict(n=-1), 1), (dict(n=0, ids=0), 0),
    (dict(vocab=0), 1), (dict(hidden=0), 1), (dict(ids=0), 1), (dict(table=0), 1), (dict(out=0), 1),
    (dict(ids=0x1004), 1), (dict(table=0x2001), 1), (dict(out=0x3002), 1), (dict(table_stride=63), 1),
    (dict(out_stride=63), 1), (dict(dtype=3), 1),                                  # no scales
    (dict(dtype=3, scales=0x4000, scales_stride=1), 1), (dict(dtype=3, scales=0x4000, scales_stride=2, table_stride=34), 1)])
def test_embedding_argument_errors(lib, kw, code):  # noqa: F811
    from lps import _lib
    a = _lib.EmbeddingArgs()
    a.ids, a.table, a.out = 0x1000, 0x2000, 0x3000
    a.id_bytes, a.dtype, a.out_dtype, a.n, a.vocab, a.hidden = 8, 1, 0, 3, 10, 64
    a.table_stride = a.out_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.lps_embedding(ctypes.byref(a), None) == code
    assert lib.lps_embedding(None, None) == 1


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 2), (dict(out_dtype=3), 2), (dict(id_bytes=1), 1), (dict(n=-1), 1), (dict(vocab=0), 1),
    (dict(n=(1 << 30) + 1), 1), (dict(hidden=0), 1), (dict(n=0, accumulate=1, out=0), 0), (dict(ids=0), 1), (dict(grad=0), 1),
    (dict(out=0), 1), (dict(ids=0x1004), 1), (dict(grad=0x2001), 1), (dict(out=0x3002), 1), (dict(grad_stride=63), 1),
    (dict(out_stride=63), 1), (dict(workspace=0), 4), (dict(workspace_bytes=16), 4), (dict(workspace=0x4008), 1)])
def test_embedding_grad_argument_errors(lib, kw, code):  # noqa: F811
    from lps import _lib
    a = _lib.EmbeddingGradArgs()
    a.ids, a.grad, a.out, a.workspace = 0x1000, 0x2000, 0x3000, 0x4000
    a.id_bytes, a.dtype, a.out_dtype, a.n, a.vocab, a.hidden = 8, 1, 0, 3000, 10, 64
    a.grad_stride = a.out_stride = 64
    a.workspace_bytes = lib.lps_embedding_grad_workspace_bytes(3000, 10, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.lps_embedding_grad(ctypes.byref(a), None) == code
    assert lib.lps_embedding_grad(None, None) == 1


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), 2), (dict(out_dtype=3), 2), (dict(rows=-1), 1), (dict(rows=0, x=0), 0), (dict(vocab=0), 1),
    (dict(hidden=0), 1), (dict(vocab=(1 << 21) + 1), 1), (dict(hidden=(1 << 24) + 1), 1),
    (dict(x_stride=(1 << 22) + 8), 1), (dict(w_stride=(1 << 23) + 16), 1), (dict(x=0), 1), (dict(w=0), 1),
    (dict(w_scales=0), 1), (dict(out=0), 1), (dict(x=0x1008), 1), (dict(x_stride=100), 1), (dict(x_stride=96), 1),
    (dict(w=0x2008), 1), (dict(w_stride=48), 1), (dict(w_stride=72), 1),
    (dict(w_scales=0x3002), 1), (dict(w_scales_stride=6), 1), (dict(w_scales_stride=0), 1), (dict(out_stride=9), 1),
    (dict(dtype=3, x_stride=64), 1),                                                  # 4-bit x without scales
    (dict(dtype=3, x_stride=56, x_scales=0x5000, x_scales_stride=4), 1),
    (dict(dtype=3, x_stride=64, x_scales=0x5000, x_scales_stride=5), 1),
    (dict(dtype=3, x_stride=64, x_scales=0x5001, x_scales_stride=4), 1)])
def test_lm_head_mx4_argument_errors(lib, kw, code):  # noqa: F811
    from lps import _lib
    a = _lib.LmHeadMx4Args()
    a.x, a.w, a.w_scales, a.out = 0x1000, 0x2000, 0x3000, 0x4000
    a.dtype, a.out_dtype, a.rows, a.vocab, a.hidden = 1, 0, 3, 10, 97
    a.x_stride, a.w_stride, a.w_scales_stride, a.out_stride = 104, 64, 4, 10
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.lps_lm_head_mx4(ctypes.byref(a), None) == code
    assert lib.lps_lm_head_mx4(None, None) == 1


def test_workspace_bytes(lib):  # noqa: F811
    f = lib.lps_embedding_grad_workspace_bytes
    assert f(-1, 10, 10) == f(3, 0, 10) == f(3, 10, 0) == 0
    assert f(0, 10, 10) == f(768, 151936, 4096) == 0              # few positions: no workspace
    assert 0 < f(769, 10, 10) <= f(2049, 10, 1000) <= f(100000, 10, 1000)
    assert f(5, 1 << 30, 8) > 0


def test_cpu_tensors_are_refused():
    import lps
    x, ids = torch.zeros((2, 32)), torch.zeros((2,), dtype=torch.int64)
    t = lps.Mx4Tensor(torch.zeros((2, 16), dtype=torch.uint8), torch.ones((2, 1), dtype=torch.uint8), 32)
    assert t.shape == (2, 32)
    for call in (lambda: lps.lm_head(x.bfloat16(), t), lambda: lps.mx4_quantize(x), lambda: lps.mx4_dequantize(t), lambda: lps.embedding(ids, x),
                 lambda: lps.embedding(ids, t), lambda: lps.embedding_grad(ids, x, 4)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
