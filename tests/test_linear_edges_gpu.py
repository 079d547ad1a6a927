"""Linear attention and layer norm where a call could be answered without an error and wrongly."""

import pytest
import torch
from torch.autograd import forward_ad

from lm_engine_amd import chunk_linear_attention, fused_recurrent_linear_attention, layer_norm
from tests.test_linear_attention_gpu import _cuda, _inputs


pytestmark = pytest.mark.gpu


def _dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
@pytest.mark.parametrize("fn", [chunk_linear_attention, fused_recurrent_linear_attention], ids=lambda f: f.__name__)
def test_tangents_are_refused_by_linear_attention(fn, grad):
    """No forward-mode derivative: a result without a tangent would read as one of zero."""
    inputs = _cuda(_inputs(2, 70, 2, 64, 64))
    want = fn(**inputs)[0]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert torch.equal(fn(**inputs)[0], want)  # (no operand has one)
        for name in inputs:
            with pytest.raises(NotImplementedError):
                fn(**{**inputs, name: _dual(inputs[name])})
    state, before = inputs["initial_state"], inputs["initial_state"].clone()
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
        fused_recurrent_linear_attention(**{**inputs, "q": _dual(inputs["q"])}, output_final_state=True, inplace_state=True)
    assert torch.equal(state, before)
    q = inputs["q"].requires_grad_()
    o, final = fn(**inputs, output_final_state=True)
    with forward_ad.dual_level():  # the gradient's tangent, by that of the output's gradient
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(o, q, _dual(torch.ones_like(o)), retain_graph=True)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad((o, final), q, (torch.ones_like(o), _dual(torch.ones_like(final))), retain_graph=True)
    assert torch.autograd.grad(o, q, torch.ones_like(o))[0].isfinite().all()


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
def test_tangents_are_refused_by_layer_norm(grad):
    x, w, b = torch.randn(5, 96, device="cuda"), torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    want = layer_norm(x, w, b)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        assert torch.equal(layer_norm(x, w, b), want)
        for i in range(3):
            with pytest.raises(NotImplementedError):
                layer_norm(*[_dual(t) if i == j else t for j, t in enumerate((x, w, b))])
    x.requires_grad_()
    y = layer_norm(x, w, b)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(y, x, _dual(torch.ones_like(y)), retain_graph=True)
    assert torch.autograd.grad(y, x, torch.ones_like(y))[0].isfinite().all()
