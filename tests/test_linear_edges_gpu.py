"""Linear attention and layer norm where a call could be answered without an error and wrongly: dual tensors, decays that grow the state."""

import pytest
import torch
from torch.autograd import forward_ad

from lm_engine_amd import chunk_linear_attention, fused_recurrent_linear_attention, layer_norm
from oracle.linear_attention_oracle import linear_attention_ref
from tests.test_linear_attention_gpu import BF16, F32, OUT, STATE, _check, _check_gradients, _cu, _cuda, _gradients, _inputs


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


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens", [[5], [1], [33], [50], [5, 17, 0, 33, 3]], ids=str)
def test_a_state_that_grows(lens, dtype):
    """g = 1.5: 50 tokens grow a state by e^75, and fp32 holds it; e^89 (59 tokens) it would not.  Whatever a short chunk has in the place of
    its missing tokens must not overflow into the results.  A power w^n is off by n g 2^-24 < 5e-6 relative, inside the state's limit."""
    T, H = sum(lens) + (3 if len(lens) > 1 else 0), 2
    inputs = _inputs(1, T, H, 64, 72, N=len(lens), dtype=dtype)
    inputs["g"] = torch.tensor([1.5, 1.4])
    cu = _cu(lens) if len(lens) > 1 else None
    cu_gpu = None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda()
    want, want_state = linear_attention_ref(**inputs, cu_seqlens=cu)
    for fn in (chunk_linear_attention, fused_recurrent_linear_attention):
        o, state = fn(**_cuda(inputs), output_final_state=True, cu_seqlens=cu_gpu)
        _check("o", o, want, OUT[dtype])
        _check("state", state, want_state, STATE[dtype])
    got, expected = _gradients(inputs, dtype, learned=True, cu=cu)
    _check_gradients(got, expected, dtype)
