"""GPU tests of the mixer operators where offsets pass 2^31 elements: every sequence (row,
block of weights) is the same, so the last one has to equal the first. Inputs are expanded
views, which take no memory of their own."""

from __future__ import annotations

import pytest
import torch
from _mixertest import scan_inputs

import spikegpt_b200 as sg

pytestmark = pytest.mark.gpu

ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def test_scan_past_2_31_elements(cuda):
    """9 sequences of 2^18 steps of 1024 channels; forward, the states kept, and the
    gradients."""
    b, t, c, n = 9, 1 << 18, 1024, 4
    ins, h0, g = scan_inputs(1, 64, c, n, torch.bfloat16, cuda, seed=71)
    wide = {k: (v.repeat(1, t // 64, 1).expand(b, -1, -1) if v.ndim == 3 else v) for k, v in ins.items()}
    assert wide["x"].numel() > 2**31 and wide["x"].stride(0) == 0
    leaves = [wide[k].detach().requires_grad_() for k in ORDER]
    out, last = sg.selective_scan(*leaves, return_state=True)
    assert torch.equal(out[0], out[-1]) and torch.equal(last[0], last[-1]) and torch.isfinite(out[-1]).all()
    alone = sg.selective_scan(*[wide[k][:1] if wide[k].ndim == 3 else wide[k] for k in ORDER])
    torch.testing.assert_close(out[-1:].float(), alone.float(), rtol=2**-7, atol=1e-3)
    del alone
    cot = g.repeat(1, t // 64, 1).expand(b, -1, -1)
    grads = torch.autograd.grad(out, leaves, cot)
    for name, v in zip(ORDER, grads):
        if v.ndim == 3:
            assert torch.equal(v[0], v[-1]) and bool(v[-1, -64:].abs().sum() > 0), name


def test_convolution_past_2_31_elements(cuda):
    b, t, c = 9, 1 << 18, 1024
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(1, 64, c, generator=gen).to(cuda, torch.bfloat16).repeat(1, t // 64, 1).expand(b, -1, -1)
    w, bias = torch.randn(c, 4, generator=gen).to(cuda), torch.randn(c, generator=gen).to(cuda)
    leaf = x.detach().requires_grad_()
    y = sg.causal_conv(leaf, w, bias)
    assert y.numel() > 2**31 and torch.equal(y[0], y[-1])
    assert torch.equal(y[-1:], sg.causal_conv(x[:1], w, bias))
    (gx,) = torch.autograd.grad(y, leaf, x)
    assert torch.equal(gx[0], gx[-1]) and bool(gx[-1, -64:].abs().sum() > 0)


def test_layer_norm_past_2_31_elements(cuda):
    rows, c = 525_000, 4096
    x = torch.randn(1, c, generator=torch.Generator().manual_seed(4)).to(cuda, torch.bfloat16).expand(rows, -1)
    w = torch.rand(c, generator=torch.Generator().manual_seed(5)).to(cuda)
    leaf = x.detach().requires_grad_()
    y = sg.layer_norm(leaf, w)
    assert y.numel() > 2**31 and torch.equal(y[:1], y[-1:]) and torch.equal(y[-1:], sg.layer_norm(x[:1], w))
    assert bool((y == y[:1]).all())
    (gx,) = torch.autograd.grad(y, leaf, w.to(torch.bfloat16).expand(rows, -1))
    assert bool((gx == gx[:1]).all())


def test_4_bit_weights_past_2_31_bytes(cuda):
    k, block, blocks, g = 8192, 16384, 33, 128
    gen = torch.Generator().manual_seed(6)
    packed = torch.randint(0, 256, (block, k // 2), generator=gen, dtype=torch.uint8).to(cuda).repeat(blocks, 1)
    scales = (torch.rand(block, k // g, generator=gen) / k).to(cuda, torch.bfloat16).repeat(blocks, 1)
    assert packed.numel() > 2**31
    for dtype, m in ((torch.bfloat16, 3), (torch.bfloat16, 12), (torch.float32, 2)):
        x = torch.randn(m, k, generator=gen).to(cuda, dtype)
        y = sg.q4_linear(x, packed, scales, group_size=g)
        assert torch.equal(y[:, :block], y[:, -block:])
        torch.testing.assert_close(y[:, -block:].float(), sg.q4_linear(x, packed[:block], scales[:block],
                                                                       group_size=g).float(), rtol=2**-7, atol=1e-4)


def test_scan_step_past_2_31_states(cuda):
    b, c, n = 33, 1 << 20, 64
    state = torch.ones(b, c, n, device=cuda)
    assert state.numel() > 2**31
    x = torch.randn(1, c, generator=torch.Generator().manual_seed(7)).to(cuda, torch.bfloat16).expand(b, -1)
    B = torch.randn(1, n, generator=torch.Generator().manual_seed(8)).to(cuda, torch.bfloat16).expand(b, -1)
    A = -torch.rand(c, n, generator=torch.Generator().manual_seed(9)).to(cuda)
    y = sg.selective_scan_step_(x, x, A, B, B, state)
    assert torch.equal(y[0], y[-1]) and torch.equal(state[0], state[-1])
    assert bool((state[-1] != 1).any())
