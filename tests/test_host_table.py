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
