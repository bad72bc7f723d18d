"""The 4-bit projection of the selective model as a module: what converting the model's
type leaves of it."""

from __future__ import annotations

import copy

import pytest
import torch

from spikegpt_b200.selective_model import Q4Linear, SelectiveConfig, SelectiveLM


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16, torch.float64])
def test_scales_keep_their_type_and_values(dtype):
    torch.manual_seed(0)
    linear = torch.nn.Linear(70, 9)
    linear.weight.data[0] *= 1e-6  # scales that float16 has not
    layer = Q4Linear(linear, 32)
    weight, scales = layer.weight(), layer.scales.clone()
    for moved in (copy.deepcopy(layer).to(dtype), torch.nn.Sequential(copy.deepcopy(layer)).to(dtype=dtype)[0]):
        assert moved.scales.dtype == torch.bfloat16 and torch.equal(moved.scales, scales)
        assert torch.equal(moved.weight(), weight) and "scales" in dict(moved.named_buffers())
        assert moved.bias.dtype == dtype
        again = Q4Linear(torch.nn.Linear(70, 9), 32).to(dtype)
        again.load_state_dict(moved.state_dict())
        assert torch.equal(again.weight(), weight)
    assert layer.to("meta").scales.is_meta and layer.scales.dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float16, 1e-2), (torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
def test_a_quantized_model_in_another_type_generates(cuda, dtype, tol):
    """Rounding the rest of the model moves the logits by a handful of the type's roundings of
    their scale; the 4-bit weights are the same."""
    torch.manual_seed(1)
    model = SelectiveLM(SelectiveConfig(vocab_size=50, n_layer=2, n_embd=48)).to(cuda).quantize_(32)
    ids = torch.randint(0, 50, (2, 12), generator=torch.Generator().manual_seed(0)).to(cuda)
    want, states = model.prefill(ids)
    next_want = model.step(ids[:, 0], states)
    other = copy.deepcopy(model).to(dtype)
    got, states = other.prefill(ids)
    assert got.dtype == dtype
    assert float((got.float() - want).abs().max()) <= tol * float(want.abs().max())
    step = other.step(ids[:, 0], states)
    assert float((step.float() - next_want).abs().max()) <= tol * float(next_want.abs().max())
