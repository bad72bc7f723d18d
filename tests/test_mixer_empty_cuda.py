"""GPU tests of the selective-mixer operators without channels, sequences, steps or rows:
every output and gradient that exists is written."""

from __future__ import annotations

import pytest
import torch
from _mixertest import scan_inputs

import spikegpt_b200 as sg
from spikegpt_b200 import _capi

pytestmark = pytest.mark.gpu

ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
def test_scan_backward_without_channels_writes_its_sums(cuda, dtype, code):
    b, t, n = 2, 37, 16
    held = torch.full((2, b * t * n + 8), float("nan"), dtype=dtype, device=cuda)
    gB, gC = held[0, : b * t * n], held[1, : b * t * n]
    row = [t * n, n]
    assert _capi.lib().selective_scan_backward(
        code, None, None, None, None, gB.data_ptr(), gC.data_ptr(), None, None, None, None, None, None, None, None, None,
        gB.data_ptr(), gC.data_ptr(), None, None, None, None, None, 0, b, t, 0, n, 0, 0, 0, 0, 0, 0, *row, *row, 0, 0, 1,
        torch.cuda.current_stream().cuda_stream) == 0  # fmt: skip
    assert (gB == 0).all() and (gC == 0).all() and held[:, b * t * n :].isnan().all()


@pytest.mark.parametrize("b,t,c", [(2, 37, 0), (0, 37, 24), (2, 0, 24), (0, 0, 0)])
def test_empty_calls_have_zero_gradients(cuda, b, t, c):
    ins, h0, g = scan_inputs(b, t, c, 16, torch.float32, cuda)
    leaves = [ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    spoil = [torch.full((b * t * 16 + 1,), float("nan"), device=cuda) for _ in range(4)]
    del spoil  # what the allocator hands out next is not zeros by chance
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True)
    assert out.shape == (b, t, c) and last.shape == (b, c, 16)
    for name, leaf, v in zip((*ORDER, "initial_state"), leaves, torch.autograd.grad(out, leaves, g)):
        assert v.shape == leaf.shape and (v == 0).all(), name
    x, w, bias = torch.randn(b, t, c, device=cuda), torch.randn(c, 4, device=cuda), torch.randn(c, device=cuda)
    leaves = [v.requires_grad_() for v in (x, w, bias)]
    for v in torch.autograd.grad(sg.causal_conv(*leaves).sum(), leaves):
        assert (v == 0).all()
