"""CPU tests of the selective-mixer operators' host side: the 4-bit format's round
trip, refusals without a GPU, the C ABI's argument checks (no launches), and the
size queries."""

from __future__ import annotations

import ctypes

import pytest
import torch

import spikegpt_b200 as sg
from spikegpt_b200 import _capi
from spikegpt_b200.selective import _kept_bytes


@pytest.mark.parametrize("k,g", [(64, 64), (100, 32), (1, 32), (75, 64), (256, 96)])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantize_round_trip(k, g, symmetric):
    """A weight comes back within half a step of its group, and a little more where the
    bfloat16 rounding of the scale (2^-9 of 15 steps) or of the zero point's integer
    moves the grid's end."""
    w = torch.randn(13, k, generator=torch.Generator().manual_seed(k))
    packed, scales, zeros = sg.quantize_q4(w, g, symmetric=symmetric)
    groups = -(-k // g)
    assert packed.shape == (13, -(-k // 32) * 16) and packed.dtype == torch.uint8
    assert scales.shape == (13, groups) and scales.dtype == torch.bfloat16
    assert (zeros is None) == symmetric
    back = sg.dequantize_q4(packed, scales, zeros, k, g)
    step = scales.float().repeat_interleave(g, 1)[:, :k]
    assert ((back - w).abs() <= (1.0 + 15 * 2**-8) * step + 1e-12).all()
    assert ((back - w).abs() <= 0.55 * step).float().mean() > 0.9


def test_quantize_zero_and_one_sided_groups():
    w = torch.zeros(2, 64)
    w[1, :32] = torch.linspace(0.5, 1.0, 32)
    for symmetric in (False, True):
        packed, scales, zeros = sg.quantize_q4(w, 32, symmetric=symmetric)
        back = sg.dequantize_q4(packed, scales, zeros, 64, 32)
        assert (back[0] == 0).all() and (back[1, 32:] == 0).all()
        assert (back[1, :32] - w[1, :32]).abs().max() <= 0.1


def test_refusals_without_a_gpu():
    x = torch.zeros(1, 4, 8)
    with pytest.raises(NotImplementedError):
        sg.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(NotImplementedError):
        sg.selective_scan(x, x, torch.zeros(8, 2), x[..., :2], x[..., :2])
    with pytest.raises(NotImplementedError):
        sg.layer_norm(x)
    with pytest.raises(NotImplementedError):
        sg.q4_linear(x[0], *sg.quantize_q4(torch.zeros(4, 8), 32), group_size=32)
    for bad in (dict(group_size=33), dict(group_size=16)):
        with pytest.raises(ValueError):
            sg.quantize_q4(torch.zeros(4, 64), **bad)
    with pytest.raises(ValueError):
        sg.quantize_q4(torch.zeros(4))


def test_c_abi_rejects_bad_arguments_before_any_launch():
    lib, null, p = _capi.lib(), None, ctypes.c_void_p(1 << 20)  # never dereferenced
    bad = _capi.WKV_ERR_INVALID_ARGUMENT
    assert lib.causal_conv_forward(7, p, p, null, null, null, p, null, 1, 4, 8, 4, 32, 8, 1, null) == bad
    assert lib.causal_conv_forward(0, p, p, null, null, null, p, null, 1, 4, 8, 0, 32, 8, 1, null) == bad
    assert lib.causal_conv_forward(0, p, p, null, null, null, p, null, -1, 4, 8, 4, 32, 8, 1, null) == bad
    assert lib.causal_conv_forward(0, null, p, null, null, null, p, null, 1, 4, 8, 4, 32, 8, 1, null) == bad
    assert "null" in _capi.last_error()
    small = _capi.WKV_ERR_WORKSPACE_TOO_SMALL
    assert lib.causal_conv_backward(0, p, p, p, null, null, null, p, p, null, null, p, 0, 1, 4, 8, 4, 32, 8, 32, 8, 1,
                                    null) == small
    strides = [32, 8, 32, 8, 8, 2, 8, 2, 0, 0]
    fwd = [p, p, p, p, p, null, null, null, null, null, p, null]
    assert lib.selective_scan_forward(0, *fwd, null, 0, null, 0, 1, 4, 8, 0, *strides, 1, null) == bad
    assert lib.selective_scan_forward(0, *fwd, null, 0, null, 0, 1, 4, 8, 65, *strides, 1, null) == bad
    assert lib.selective_scan_forward(0, *fwd, p, 1, null, 0, 1, 4, 8, 2, *strides, 1, null) == small
    assert lib.selective_scan_step(9, p, p, p, p, p, p, null, null, null, p, 1, 8, 2, 8, 8, 2, 2, 0, 1, null) == bad
    assert lib.layer_norm_forward(0, p, null, null, p, p, p, 4, 16385, 16385, 1e-5, null) == bad
    assert lib.layer_norm_backward(0, p, p, null, p, p, p, p, p, p, 8, 4, 64, 64, 64, null) == small
    assert lib.q4_matvec(0, p, p, p, null, null, p, 1, 8, 64, 33, 64, null) == bad
    assert lib.q4_matvec(0, null, p, p, null, null, p, 1, 8, 64, 64, 64, null) == bad


def test_empty_calls_do_nothing():
    lib, null = _capi.lib(), None
    assert lib.causal_conv_forward(1, null, null, null, null, null, null, null, 0, 4, 8, 4, 32, 8, 1, null) == 0
    assert lib.layer_norm_forward(1, null, null, null, null, null, null, 0, 64, 64, 1e-5, null) == 0
    assert lib.q4_matvec(1, null, null, null, null, null, null, 0, 8, 64, 64, 64, null) == 0


def test_size_queries():
    lib = _capi.lib()
    for b, t, c, n in ((1, 1, 1, 1), (2, 17, 33, 16), (3, 1024, 512, 64), (2, 0, 4, 4)):
        assert lib.selective_scan_state_size(b, t, c, n) == _kept_bytes(b, t, c, n)
    assert lib.causal_conv_workspace_size(2, 100, 64, 5) == 0  # an invalid width
    assert lib.layer_norm_workspace_size(0, 0, 64) == 0


def test_selective_model_builds_and_quantizes_on_the_cpu():
    from spikegpt_b200.selective_model import Q4Linear, SelectiveConfig, SelectiveLM

    with pytest.raises(ValueError):
        SelectiveLM(SelectiveConfig(n_state=65))
    with pytest.raises(ValueError):
        SelectiveLM(SelectiveConfig(taps=5))
    model = SelectiveLM(SelectiveConfig(vocab_size=33, n_layer=2, n_embd=24, n_state=4))
    assert model.blocks[0].in_proj.weight.shape == (96, 24) and model.blocks[0].A_log.shape == (48, 4)
    head = model.head.weight.detach().clone()
    model.quantize_(32)
    assert isinstance(model.head, Q4Linear) and model.head.weight().shape == head.shape
    assert (model.head.weight() - head).abs().max() <= 0.1 * head.abs().max()
    again = SelectiveLM(SelectiveConfig(vocab_size=33, n_layer=2, n_embd=24, n_state=4)).quantize_(32)
    again.load_state_dict(model.state_dict())
    assert torch.equal(again.head.weight(), model.head.weight())
