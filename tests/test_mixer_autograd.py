"""CPU tests of what the mixer operators tell autograd, on meta tensors: derivatives that
they do not have raise instead of being dropped."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import spikegpt_b200 as sg

B, T, C, N, W = 2, 5, 8, 4, 4
PACKED = sg.quantize_q4(torch.zeros(3, C), 32)


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="meta")


def _inputs():
    packed, scales, points = (v.to("meta") for v in PACKED)
    one = dict(x=zeros(B, C), dt=zeros(B, C), A=zeros(C, N), B=zeros(B, N), C=zeros(B, N), state=zeros(B, C, N),
               D=zeros(C), z=zeros(B, C), dt_bias=zeros(C))
    return {
        "layer_norm": (sg.layer_norm, dict(x=zeros(B, C), weight=zeros(C), bias=zeros(C))),
        "causal_conv": (sg.causal_conv, dict(x=zeros(B, T, C), weight=zeros(C, W), bias=zeros(C),
                                             initial_state=zeros(B, W - 1, C))),
        "selective_scan": (sg.selective_scan, dict(
            x=zeros(B, T, C), dt=zeros(B, T, C), A=zeros(C, N), B=zeros(B, T, N), C=zeros(B, T, N), D=zeros(C),
            z=zeros(B, T, C), dt_bias=zeros(C), initial_state=zeros(B, C, N))),
        "causal_conv_step_": (sg.causal_conv_step_, dict(x=zeros(B, C), state=zeros(B, W - 1, C), weight=zeros(C, W),
                                                         bias=zeros(C))),
        "selective_scan_step_": (sg.selective_scan_step_, one),
        "q4_linear": (sg.q4_linear, dict(x=zeros(B, C), packed=packed, scales=scales, zeros=points, bias=zeros(3),
                                         group_size=32)),
    }  # fmt: skip


CASES = [(op, name) for op, (_, args) in _inputs().items() for name, v in args.items()
         if isinstance(v, torch.Tensor) and v.is_floating_point()]  # fmt: skip
NO_GRADIENT = ("causal_conv_step_", "selective_scan_step_", "q4_linear")


@pytest.mark.parametrize("op,name", CASES)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(op, name, grad_mode):
    f, args = _inputs()[op]
    with fwAD.dual_level(), torch.set_grad_enabled(grad_mode), pytest.raises(NotImplementedError, match="forward-mode"):
        f(**{**args, name: fwAD.make_dual(args[name], torch.ones_like(args[name]))})
    with torch.set_grad_enabled(grad_mode), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: f(**{**args, name: v}), (args[name],), (args[name],))
    with fwAD.dual_level():  # a level without tangents is no reason to refuse
        f(**args)


@pytest.mark.parametrize("op,name", [c for c in CASES if c[0] in NO_GRADIENT])
def test_operators_without_a_gradient_refuse_every_route_to_one(op, name):
    f, args = _inputs()[op]
    with pytest.raises(NotImplementedError, match="no gradient"):
        f(**{**args, name: args[name].requires_grad_()})
    f, args = _inputs()[op]
    with pytest.raises(NotImplementedError, match="no gradient"):
        torch.func.grad(lambda v: f(**{**args, name: v}).sum())(args[name])
    with pytest.raises(NotImplementedError, match="no gradient"):
        torch.func.vjp(lambda v: f(**{**args, name: v}), args[name])
    with torch.no_grad():
        f(**{**args, name: args[name].requires_grad_()})


@pytest.mark.parametrize("op", ["layer_norm", "causal_conv", "selective_scan"])
def test_function_transforms_do_not_lose_a_gradient(op):
    f, args = _inputs()[op]
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: f(**{**args, "x": v}).sum())(args["x"])


@pytest.mark.parametrize("op", ["causal_conv_step_", "selective_scan_step_"])
def test_steps_say_that_they_write_in_place(op):
    f, args = _inputs()[op]
    holder = zeros(2, *args["state"].shape)
    for state in (args["state"], holder[1]):
        before = state._version
        f(**{**args, "state": state})
        assert state._version == before + 1
    assert holder._version == 1
    with torch.no_grad():
        f(**args)
    assert args["state"]._version == 2
    with pytest.raises(ValueError):
        f(**{**args, "x": args["x"][:1]})
    with torch.inference_mode():
        held = zeros(*args["state"].shape)
        f(**{**args, "state": held})
    with torch.no_grad():
        f(**{**args, "state": held})


def test_a_step_on_a_saved_window_is_noticed():
    """causal_conv saves its initial window; a step on that window before the backward
    would give other gradients."""
    weight = zeros(C, W).requires_grad_()
    window = zeros(B, W - 1, C)
    y = sg.causal_conv(zeros(B, T, C), weight, initial_state=window)
    y.sum().backward(retain_graph=True)
    with torch.no_grad():
        sg.causal_conv_step_(zeros(B, C), window, weight)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


DIFFERENTIABLE = [c for c in CASES if c[0] not in NO_GRADIENT]
LINEAR = [("layer_norm", "bias"), ("selective_scan", "initial_state")]  # their gradients do not depend on them


@pytest.mark.parametrize("op,name", DIFFERENTIABLE)
def test_second_derivatives_are_refused(op, name):
    """With create_graph the gradients can be used, and differentiating them raises: a
    gradient penalty must not train on nothing."""
    f, args = _inputs()[op]
    leaf = args[name].requires_grad_()
    y = f(**args)
    (grad,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    assert grad.requires_grad == ((op, name) not in LINEAR) and grad.shape == leaf.shape
    if grad.requires_grad:
        with pytest.raises((RuntimeError, NotImplementedError), match="not implemented"):
            grad.sum().backward()
    y = f(**args)
    cotangent = zeros(*y.shape).requires_grad_()
    (grad,) = torch.autograd.grad(y, leaf, cotangent, create_graph=True)
    with pytest.raises((RuntimeError, NotImplementedError), match="not implemented"):
        torch.autograd.grad(grad.sum(), cotangent)
    y = f(**args)
    assert not torch.autograd.grad(y.sum(), leaf)[0].requires_grad


@pytest.mark.parametrize("op", ["layer_norm", "causal_conv", "selective_scan"])
def test_tangents_of_a_gradient_are_refused(op):
    f, args = _inputs()[op]
    x = args["x"].requires_grad_()
    y = f(**args)
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(y, x, fwAD.make_dual(zeros(*y.shape), zeros(*y.shape)))
    if op == "selective_scan":  # its gradients come as a list, which has no batched form
        return
    y = f(**args)
    (many,) = torch.autograd.grad(y, x, zeros(3, *y.shape), is_grads_batched=True)
    assert many.shape == (3, *x.shape)
