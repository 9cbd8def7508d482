"""The autograd form of the gated block around a stand-in for its launches: which calls keep the products, and which derivatives it refuses.
No GPU is touched."""

import pytest
import torch
from torch.autograd import forward_ad

from cppmega_mlx_amd.nn import gated_ffn as gf


@pytest.fixture
def kept(monkeypatch):
    """The stand-in's calls: the type of the kept products, or None."""
    calls = []

    def block(x, w, offsets=None, *, activation="silu", out=None, pre=None):
        calls.append(None if pre is None else pre.dtype)
        p = x.detach() @ w.detach().T
        if pre is not None:
            pre.copy_(p)
        g, u = p.chunk(2, -1)
        return torch.nn.functional.silu(g) * u

    monkeypatch.setattr(gf, "gated_gemm", block)
    return calls


def _operands():
    g = torch.Generator().manual_seed(1)
    return torch.randn(3, 5, generator=g, dtype=torch.float64), torch.randn(8, 5, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("which", ["x", "w", "both"])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("wanted", [True, False])
def test_forward_mode_derivatives_are_refused(kept, which, grad, wanted):
    """A result without its tangent would be taken for a constant by all that follows."""
    x, w = _operands()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        a = x if which == "w" else forward_ad.make_dual(x, torch.ones_like(x))
        b = w if which == "x" else forward_ad.make_dual(w, torch.ones_like(w))
        if wanted and which != "both":
            (b if which == "x" else a).requires_grad_()
        with pytest.raises(RuntimeError, match="jvp"):
            gf.gated_gemm_apply(a, b)


def test_function_transforms_are_refused(kept):
    x, w = _operands()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: gf.gated_gemm_apply(t, w), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: gf.gated_gemm_apply(t, w))(x.expand(2, 3, 5))


def test_products_are_kept_where_a_gradient_is_wanted(kept):
    x, w = _operands()
    plain = gf.gated_gemm_apply(x, w)
    assert kept == [None] and not plain.requires_grad
    w.requires_grad_()
    with torch.no_grad():
        assert not gf.gated_gemm_apply(x, w).requires_grad
    with torch.inference_mode():
        gf.gated_gemm_apply(x, w)
    assert kept == [None] * 3
    y = gf.gated_gemm_apply(x, w, pre_dtype=torch.float64)
    assert kept[3:] == [torch.float64] and y.requires_grad and torch.equal(y, plain)
