"""GPU tests of the single-token steps and the 4-bit product under torch.compile, and of
the vectorising transform, against eager calls."""

from __future__ import annotations

import pytest
import torch
from _mixertest import scan_inputs

import spikegpt_b200 as sg

pytestmark = pytest.mark.gpu


def _token(device, b=3, c=48, n=16, seed=51):
    ins, h0, _ = scan_inputs(b, 1, c, n, torch.bfloat16, device, seed=seed)
    one = {k: (v[:, 0] if v.ndim == 3 else v) for k, v in ins.items()}
    gen = torch.Generator().manual_seed(seed)
    window = torch.randn(b, 3, c, generator=gen).to(device, torch.bfloat16)
    weight, bias = torch.randn(c, 4, generator=gen).to(device), torch.randn(c, generator=gen).to(device)
    packed = sg.quantize_q4(torch.randn(33, c, generator=gen).to(device), 32)
    return one, h0, window, weight, bias, packed


def test_steps_and_4_bit_product_compile_fullgraph(cuda):
    """One graph without breaks, whose calls move the window and the state on in place."""
    one, h0, window, weight, bias, packed = _token(cuda)

    def token(x, window, state):
        u = sg.causal_conv_step_(x, window, weight, bias)
        y = sg.selective_scan_step_(u, one["dt"], one["A"], one["B"], one["C"], state, one["D"], one["z"],
                                    one["dt_bias"])
        return sg.q4_linear(sg.layer_norm(y, bias), *packed, group_size=32)

    compiled = torch.compile(token, fullgraph=True)
    a, b = (window.clone(), h0.clone()), (window.clone(), h0.clone())
    with torch.no_grad():
        for i in range(3):
            x = one["x"] * (1 + i)
            want, got = token(x, *a), compiled(x, *b)
            torch.testing.assert_close(got, want, rtol=2**-6, atol=2**-6)
            assert torch.equal(a[0], b[0])
            torch.testing.assert_close(b[1], a[1], rtol=1e-5, atol=1e-6)


def test_vmap_is_a_loop_over_calls(cuda):
    one, _, _, weight, bias, packed = _token(cuda)
    x = torch.randn(4, 2, 9, 48, generator=torch.Generator().manual_seed(1)).to(cuda, torch.bfloat16)
    for f in (lambda v: sg.layer_norm(v, bias), lambda v: sg.causal_conv(v, weight, bias),
              lambda v: sg.q4_linear(v, *packed, group_size=32)):  # fmt: skip
        assert torch.equal(torch.vmap(f)(x), torch.stack([f(v) for v in x]))


def test_gradients_recorded_for_a_graph_of_gradients_are_the_same(cuda):
    ins, _, g = scan_inputs(2, 30, 40, 16, torch.float32, cuda, seed=53)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    leaves = [ins[k].requires_grad_() for k in names]

    def loss():
        u = sg.causal_conv(leaves[0], weight, leaves[7])
        return (sg.layer_norm(sg.selective_scan(u, *leaves[1:]), leaves[5]) * g).sum()

    weight = torch.randn(40, 4, generator=torch.Generator().manual_seed(2)).to(cuda).requires_grad_()
    plain = torch.autograd.grad(loss(), [*leaves, weight])
    recorded = torch.autograd.grad(loss(), [*leaves, weight], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, recorded))
    with pytest.raises((RuntimeError, NotImplementedError), match="not implemented"):
        sum((v * v).sum() for v in recorded).backward()
