"""The vocabulary table's host layer (CPU, no GPU): what its calls do about
derivatives, outputs and operands, with plain torch in the kernels' place."""

import pytest
import torch
from torch.autograd import forward_ad

import lps
from lps import vocab_table as T


@pytest.fixture
def plain_lookup(monkeypatch):
    """The lookup and its gradient by torch's own indexing."""
    def lookup(ids, table, scale, out_dtype):
        valid = (ids >= 0) & (ids < table.shape[0])
        rows = table.detach().float()[torch.where(valid, ids, 0)] * scale
        return torch.where(valid[..., None], rows, 0.0).to(out_dtype or table.dtype)
    monkeypatch.setattr(T, "_embedding", lookup)


IDS = torch.tensor([[0, 4, -1], [2, 4, 9]])


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, None), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangent_of_a_lookup(plain_lookup, dtype, out_dtype, grad_mode):
    """A dual table's tangent comes out as its own lookup, with or without reverse mode."""
    g = torch.Generator().manual_seed(1)
    w, t = torch.randn((5, 8), generator=g).to(dtype), torch.randn((5, 8), generator=g).to(dtype)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        out = forward_ad.unpack_dual(lps.embedding(IDS, forward_ad.make_dual(w, t), scale=3.0, out_dtype=out_dtype))
        assert torch.equal(out.primal, T._embedding(IDS, w, 3.0, out_dtype))
        assert out.tangent is not None and torch.equal(out.tangent, T._embedding(IDS, t, 3.0, out_dtype))
        # a table without a tangent inside the level
        assert forward_ad.unpack_dual(lps.embedding(IDS, w)).tangent is None
        both = lps.embedding(IDS, forward_ad.make_dual(w.clone().requires_grad_(), t))
        assert both.requires_grad == grad_mode and forward_ad.unpack_dual(both).tangent is not None


@pytest.fixture
def anywhere(monkeypatch):
    """CPU tensors pass for the GPU's; the entry points' calls are kept, not made."""
    from lps import lmhead
    calls = []
    for m in (T, lmhead):
        monkeypatch.setattr(m, "_on_gpu", lambda t, name: None)
        monkeypatch.setattr(m, "_call", lambda name, args, device: calls.append((name, args)))
    return calls


def _weight(V, H):
    n = -(-H // 32)
    return lps.Mx4Tensor(torch.zeros((V, 16 * n), dtype=torch.uint8), torch.full((V, n), 127, dtype=torch.uint8), H)


def test_derivatives_that_a_call_does_not_have(anywhere):
    """An input that asks for one is refused, not answered without it; the same call
    without gradients, or of a detached input, is made."""
    w = _weight(8, 64)
    x, grad, out = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((2, 64)), torch.zeros((8, 64))
    ids = torch.tensor([1, 3])
    cases = [(x, lambda t: lps.lm_head(t, w)), (x, lambda t: lps.lm_head(t, w, return_stats=True)),
             (grad, lambda t: lps.embedding_grad(ids, t, 8)), (out, lambda t: lps.embedding_grad(ids, grad, 8, out=t))]
    for t, call in cases:
        needs = t.clone().requires_grad_()
        with pytest.raises(ValueError, match="derivative|gradient"):
            call(needs)
        with forward_ad.dual_level(), pytest.raises(ValueError, match="derivative"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
        assert not anywhere
        with torch.no_grad():
            call(needs)
        call(needs.detach())
        with forward_ad.dual_level():
            call(t)
        assert len(anywhere) == 3
        anywhere.clear()


def test_tangent_of_a_lookups_gradient(plain_lookup, anywhere):
    """Forward over reverse is refused too."""
    w = torch.ones((5, 8)).requires_grad_()
    with forward_ad.dual_level(), pytest.raises(ValueError, match="derivative"):
        out = lps.embedding(IDS, forward_ad.make_dual(w, torch.ones((5, 8))))
        (out * out).sum().backward()


def test_quantised_values_have_no_gradient(anywhere):
    """Codes and scales are whole numbers: a weight that requires a gradient is quantised without one."""
    t = lps.mx4_quantize(torch.nn.Parameter(torch.ones((4, 40))))
    assert not t.codes.requires_grad and not t.scales.requires_grad and len(anywhere) == 1


def test_out_counts_as_written(anywhere):
    """A graph that saved out must not use the changed values."""
    ids, grad, out = torch.tensor([1, 3]), torch.zeros((2, 8)), torch.ones((4, 8))
    w = torch.ones((4, 8)).requires_grad_()
    loss = (w * out).sum()                            # saves out
    lps.embedding_grad(ids, grad, 4, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    view = torch.ones((4, 20))
    before = view._version
    lps.embedding_grad(ids, grad, 4, out=view[:, 3:11])
    assert view._version > before
    with torch.inference_mode():
        lps.embedding_grad(ids, grad, 4, out=torch.ones((4, 8)))


def _bytes_of(t):
    """Every byte address that t's elements take."""
    at = [t.data_ptr()]
    for n, s in zip(t.shape, t.stride()):
        at = [a + i * s * t.element_size() for a in at for i in range(n)]
    return {a + k for a in at for k in range(t.element_size())}


def test_out_that_shares_memory_with_its_inputs(anywhere):
    """Refused where a byte is shared, and only there: rows between each other's are two tensors."""
    buf = torch.zeros(4096)
    sizes = [(1, 8, 8), (4, 8, 8), (4, 8, 20), (5, 3, 20), (3, 8, 28), (6, 5, 9), (4, 12, 20)]
    seen = set()
    for V, H, s in sizes:
        out = buf[200:].as_strided((V, H), (s, 1))
        for n, h, t in sizes:
            if h != H:
                continue
            for off in range(120, 360, 4):
                grad = buf[off:].as_strided((n, H), (t, 1))
                shared = bool(_bytes_of(out) & _bytes_of(grad))
                between = not shared and off < 200 + V * s and off + n * t > 200
                seen.add((shared, between))
                call = lambda: lps.embedding_grad(torch.zeros(n, dtype=torch.int64), grad, V, out=out)  # noqa: E731
                if shared:
                    with pytest.raises(ValueError, match="overlap"):
                        call()
                else:
                    call()
    assert seen == {(True, False), (False, False), (False, True)}
    half = buf.view(torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        lps.embedding_grad(torch.tensor([0, 1]), half[:16].view(2, 8), 4, out=buf[:32].view(4, 8))
    ids = buf.view(torch.int64)[:4]
    with pytest.raises(ValueError, match="overlap"):
        lps.embedding_grad(ids, torch.zeros((4, 8)), 4, out=buf[6:38].view(4, 8))
    lps.embedding_grad(ids, torch.zeros((4, 8)), 4, out=buf[8:40].view(4, 8))
    # a gradient that is copied first (every position the same row) is read before out is written
    lps.embedding_grad(torch.zeros(3, dtype=torch.int64), buf[:8].expand(3, 8), 4, out=buf[:32].view(4, 8))
    lps.embedding_grad(torch.zeros(0, dtype=torch.int64), buf[:0].view(0, 8), 4, out=buf[:32].view(4, 8))


def _strided(V, n, s):
    """uint8 [V, n], rows s bytes apart."""
    return torch.zeros((V - 1) * s + n, dtype=torch.uint8).as_strided((V, n), (s, 1))


@pytest.mark.parametrize("M,H,xs,dtype", [
    (3, 1 << 22, 1 << 22, torch.bfloat16), (3, (1 << 22) + 8, (1 << 22) + 8, torch.float16),
    (2, (1 << 22) + 3, (1 << 22) + 3, torch.bfloat16), (2, 64, (1 << 22) + 8, torch.bfloat16),
    (2, 64, (1 << 23) + 16, "mx4"), (3, 64, 32, "mx4"), (1, (1 << 24), 1 << 24, torch.bfloat16)])
@pytest.mark.parametrize("ws", [0, (1 << 23) + 16])
def test_head_rows_far_apart(anywhere, M, H, xs, dtype, ws):
    """Rows more than 8 MiB apart, by their strides or their lengths: every call is one
    that the C ABI takes, and together they are all the rows."""
    from lps import _lib
    V, n = 2, -(-H // 32)
    w = lps.Mx4Tensor(_strided(V, 16 * n, max(ws, 16 * n)), torch.full((V, n), 127, dtype=torch.uint8), H)
    if dtype == "mx4":
        x = lps.Mx4Tensor(_strided(M, 16 * n, xs), torch.full((M, n), 127, dtype=torch.uint8), H)
    else:
        x = torch.zeros((M - 1) * xs + H, dtype=dtype).as_strided((M, H), (xs, 1))
    out, stats = lps.lm_head(x, w, return_stats=True)
    assert out.shape == (M, V) and stats.shape == (M, 1, 2)
    at = 0
    for _, args in anywhere:
        a = _lib.LmHeadMx4Args.from_buffer_copy(args)
        assert a.rows == 1 or (a.x_stride * (1 if dtype == "mx4" else 2) <= 1 << 23 and a.x_stride >= (16 * n if dtype == "mx4" else H))
        assert a.x_stride % (16 if dtype == "mx4" else 8) == 0 or a.rows == 1
        assert a.w_stride <= 1 << 23 and a.x % 16 == 0 and a.w % 16 == 0
        assert a.out == out.data_ptr() + at * V * out.element_size() and a.stats == stats.data_ptr() + at * 8
        at += a.rows
    assert at == M
