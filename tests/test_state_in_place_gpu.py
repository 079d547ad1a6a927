"""A state that a decode step updates in place counts as written, as after any torch operation in place: a backward that saved it raises
instead of computing with what it has become."""

import pytest
import torch

from lm_engine_amd import chunk_gated_delta_rule, chunk_linear_attention, fused_recurrent_gated_delta_rule, fused_recurrent_linear_attention


pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class LinearAttention:
    """``wide``: a decay in float64, which the native host path leaves to the Python one."""

    @staticmethod
    def inputs(tokens, wide):
        q, k, v = (torch.randn(2, tokens, 2, 64, device="cuda").to(BF16) for _ in range(3))
        g = torch.tensor([-0.1, -0.02], device="cuda", dtype=torch.float64 if wide else torch.float32)
        return dict(q=q, k=k, v=v, g=g)

    whole, step = chunk_linear_attention, fused_recurrent_linear_attention


class DeltaRule:
    @staticmethod
    def inputs(tokens, wide):
        q, k, v = (torch.randn(2, tokens, 2, 64, device="cuda").to(BF16) for _ in range(3))
        g = -0.1 * torch.rand(2, tokens, 2, device="cuda", dtype=torch.float64 if wide else torch.float32)
        return dict(q=q, k=torch.nn.functional.normalize(k, dim=-1), v=v, g=g, beta=torch.rand(2, tokens, 2, device="cuda"))

    whole, step = chunk_gated_delta_rule, fused_recurrent_gated_delta_rule


OPERATORS = [LinearAttention, DeltaRule]


def _state():
    return torch.randn(2, 2, 64, 64, device="cuda")


@pytest.mark.parametrize("wide", [False, True], ids=["native", "python"])
@pytest.mark.parametrize("operator", OPERATORS, ids=lambda x: x.__name__)
def test_an_overwritten_state_is_noticed_by_the_backward(operator, wide):
    state = _state()
    inputs = operator.inputs(70, wide)
    q = inputs["q"].requires_grad_()
    o, _ = operator.whole(**inputs, initial_state=state)
    with torch.no_grad():
        _, out = operator.step(**operator.inputs(1, wide), initial_state=state, output_final_state=True, inplace_state=True)
    assert out is state and state._version > 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.float().sum(), q)


@pytest.mark.parametrize("wide", [False, True], ids=["native", "python"])
@pytest.mark.parametrize("operator", OPERATORS, ids=lambda x: x.__name__)
def test_what_counts_as_written(operator, wide):
    inputs = operator.inputs(1, wide)
    cache = torch.randn(3, 2, 2, 64, 64, device="cuda")
    operator.step(**inputs, initial_state=cache[1], output_final_state=True, inplace_state=True)
    assert cache._version > 0  # a slot of a cache: the cache
    state = _state()
    operator.step(**inputs, initial_state=state, output_final_state=True)
    assert state._version == 0  # read only
    with pytest.raises(ValueError):
        operator.step(**inputs, initial_state=state.transpose(0, 1), output_final_state=True, inplace_state=True)
    assert state._version == 0  # refused


@pytest.mark.parametrize("wide", [False, True], ids=["native", "python"])
@pytest.mark.parametrize("operator", OPERATORS, ids=lambda x: x.__name__)
def test_states_made_in_inference_mode(operator, wide):
    """Such a tensor has no version; it is updated all the same, once, in inference mode and behind it."""
    inputs = operator.inputs(1, wide)
    with torch.inference_mode():
        state = _state()
        start = state.clone()
        operator.step(**inputs, initial_state=state, output_final_state=True, inplace_state=True)
        _, want = operator.step(**inputs, initial_state=start, output_final_state=True)
        assert torch.equal(state, want)
    with torch.no_grad():
        _, want = operator.step(**inputs, initial_state=state, output_final_state=True)
        operator.step(**inputs, initial_state=state, output_final_state=True, inplace_state=True)
        assert torch.equal(state, want)
