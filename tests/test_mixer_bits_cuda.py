"""GPU tests that float32 tensors are worked on with float32's bits where a result does not
hide it: gates at large arguments, and sums over states of terms that cancel."""

from __future__ import annotations

import pytest
import torch

import spikegpt_b200 as sg

pytestmark = pytest.mark.gpu

# An exponential within 2^-22 of its value, a reciprocal within 2^-23, three roundings of 2^-24
# around them, and the rounding of ln(2) times the exponent, 2e-9 * 115 at the largest
# argument here: 7.7e-7 of the value.
GATE = 8 * 2.0**-23


def _check_gate(got, v):
    want = v.double() * torch.sigmoid(v.double())
    worst = ((got.double() - want).abs() / want.abs()).max()
    assert float(worst) <= GATE, float(worst)


def test_gates_keep_their_relative_accuracy_at_large_arguments(cuda):
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.linspace(-80, 80, 4001), torch.randn(4191, generator=g) * 10]).to(cuda)
    v = torch.where(v == 0, torch.ones_like(v), v)
    ones, c = torch.ones(64, device=cuda), 64
    x = v.view(1, -1, c)
    _check_gate(sg.causal_conv(x, ones[:, None]), x)
    for k in range(8):
        _check_gate(sg.causal_conv_step_(x[:, k], torch.empty(1, 0, c, device=cuda), ones[:, None]), x[:, k])
    A, zero = -torch.ones(c, 4, device=cuda), torch.zeros(1, x.shape[1], 4, device=cuda)
    one = torch.ones_like(x)
    _check_gate(sg.selective_scan(one, one, A, zero, zero, ones, x), x)  # D x silu(z)
    state = torch.zeros(1, c, 4, device=cuda)
    for k in range(8):
        _check_gate(sg.selective_scan_step_(one[:, k], one[:, k], A, zero[:, k], zero[:, k], state, ones, x[:, k]), x[:, k])
    leaf = one.clone().requires_grad_()
    (gx,) = torch.autograd.grad(sg.selective_scan(leaf, one, A, zero, zero, ones, x).sum(), leaf)
    _check_gate(gx, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gates_at_their_limits(cuda, dtype):
    """Arguments past the exponential's range, infinities and NaN."""
    v = torch.tensor([-60000.0, -500.0, -104.0, 104.0, 500.0, 60000.0, float("inf"), float("nan")], device=cuda).to(dtype)
    x = v.view(1, 1, 8)
    y = sg.causal_conv(x, torch.ones(8, 1, device=cuda))[0, 0].float()
    assert (y[:3].abs() <= 1e-30).all() and torch.equal(y[3:7], v[3:7].float()) and y[7].isnan()
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(sg.causal_conv(leaf, torch.ones(8, 1, device=cuda)).sum(), leaf)
    assert (g[0, 0, :3].abs() <= 1e-30).all() and (g[0, 0, 3:6] == 1).all() and g[0, 0, 7].isnan()


@pytest.mark.parametrize("n", [3, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("c", [33, 64])
def test_sums_over_states_keep_their_terms_last_bits(cuda, n, c):
    """Two terms that cancel but for their last bits, at many pairs of states: the gradients of
    x and dt, and of the gate through y, are what float32 leaves of them, exactly."""
    t, first, second = 40, 2.0 - 2.0**-23, -(2.0 - 2.0**-21)
    C, want = torch.zeros(1, t, n, device=cuda), first + second
    for i in range(t):
        C[0, i, i % n], C[0, i, (i + 1 + i // n) % n] = first, second
    pair = (C != 0).sum(-1)[0] == 2
    assert pair.sum() >= t // 2
    one = torch.ones(1, t, c, device=cuda)
    A, B = torch.full((c, n), -1e30, device=cuda), torch.ones(1, t, n, device=cuda)  # no memory: every step alone
    x, dt, z = (one.clone().requires_grad_() for _ in range(3))
    plain = sg.selective_scan(x, dt, A, B, C, dt_softplus=False)
    for name, v in zip(("x", "dt"), torch.autograd.grad(plain.sum(), (x, dt))):
        assert (v[0, pair] == want).all(), (name, float(v[0, pair].min()), float(v[0, pair].max()), want)
    (gz,) = torch.autograd.grad(sg.selective_scan(x, dt, A, B, C, None, z, dt_softplus=False).sum(), z)
    s = torch.sigmoid(torch.ones(()).double())
    slope = float(s * (1 + (1 - s)))
    assert float((gz[0, pair].double() / slope - want).abs().max()) <= GATE * want
