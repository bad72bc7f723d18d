"""Layer norm of any row width, forward and backward, on sm_100a.

``fused.ln_shift_mix`` covers the blocks' LayerNorm together with the token shift
(float32 rows of 128 to 1024 channels, bf16 outputs). ``layer_norm`` is the plain
one, for any width up to 16384, float32, bfloat16 and float16 rows, float32
statistics and parameters: ``y = (x - mean) * rstd * weight + bias``. The backward
sums the parameters' gradients over the rows in a fixed order.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _capi
from ._mixer import code_of, need_cuda, need_shape, on_device, parameter, ptr, rows, stream, wants_grad, workspace

MAX_WIDTH = 16384


def _forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    n, c = x.shape
    y = torch.empty((n, c), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, n), dtype=torch.float32, device=x.device)
    mean, rstd = stats.unbind(0)
    _capi.check(
        _capi.lib().layer_norm_forward(code_of("x", x), x.data_ptr(), ptr(weight), ptr(bias), y.data_ptr(),
                                       mean.data_ptr(), rstd.data_ptr(), n, c, x.stride(0), eps, stream(x)),
        "layer_norm_forward",
    )
    return y, mean, rstd


def _backward(g: Tensor, x: Tensor, weight: Tensor | None, mean: Tensor, rstd: Tensor, want_weight: bool,
              want_bias: bool) -> tuple[Tensor, Tensor, Tensor]:
    n, c = x.shape
    code = code_of("x", x)
    lib = _capi.lib()
    gx = torch.empty((n, c), dtype=x.dtype, device=x.device)
    gw = torch.empty(c if want_weight else 0, dtype=torch.float32, device=x.device)
    gb = torch.empty(c if want_bias else 0, dtype=torch.float32, device=x.device)
    nws = lib.layer_norm_workspace_size(code, n, c)
    ws = workspace(nws, x)
    _capi.check(
        lib.layer_norm_backward(code, g.data_ptr(), x.data_ptr(), ptr(weight), mean.data_ptr(), rstd.data_ptr(),
                                gx.data_ptr(), gw.data_ptr() if want_weight else None,
                                gb.data_ptr() if want_bias else None, ptr(ws), nws, n, c, g.stride(0), x.stride(0),
                                stream(x)),
        "layer_norm_backward",
    )
    return gx, gw, gb


@torch.library.custom_op("spikegpt_b200::layer_norm", mutates_args=(), device_types="cuda")
def _op(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    with on_device(x) or nullcontext():
        y, mean, rstd = _forward(rows(x), weight, bias, eps)
    return y, mean.clone(), rstd.clone()  # a custom op's outputs share no memory


@_op.register_fake
def _(x, weight, bias, eps):
    stat = x.new_empty(x.shape[0], dtype=torch.float32)
    return x.new_empty(x.shape), stat, torch.empty_like(stat)


@torch.library.custom_op("spikegpt_b200::layer_norm_backward", mutates_args=(), device_types="cuda")
def _op_backward(g: Tensor, x: Tensor, weight: Tensor | None, mean: Tensor, rstd: Tensor, want_weight: bool,
                 want_bias: bool) -> tuple[Tensor, Tensor, Tensor]:
    with on_device(x) or nullcontext():
        return _backward(rows(g), rows(x), weight, mean, rstd, want_weight, want_bias)


@_op_backward.register_fake
def _(g, x, weight, mean, rstd, want_weight, want_bias):
    c = x.shape[1]
    return (x.new_empty(x.shape), x.new_empty(c if want_weight else 0, dtype=torch.float32),
            x.new_empty(c if want_bias else 0, dtype=torch.float32))


def _setup(ctx, inputs, output):
    x, weight, bias, _eps = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.has_bias = bias is not None
    ctx.mark_non_differentiable(output[1], output[2])


def _op_grad(ctx, g, _gmean, _grstd):
    x, weight, mean, rstd = ctx.saved_tensors
    gx, gw, gb = torch.ops.spikegpt_b200.layer_norm_backward(g.to(x.dtype), x, weight, mean, rstd, weight is not None,
                                                             ctx.has_bias)
    return gx, gw if weight is not None else None, gb if ctx.has_bias else None, None


_op.register_autograd(_op_grad, setup_context=_setup)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, mean, rstd = ctx.saved_tensors
        with on_device(x) or nullcontext():
            gx, gw, gb = _backward(rows(g), x, weight, mean, rstd, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return gx, gw if ctx.needs_input_grad[1] else None, gb if ctx.needs_input_grad[2] else None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """Layer norm of ``x`` [..., C] (CUDA, float32 / bfloat16 / float16, C <= 16384)
    over its last dimension, in x's dtype; weight and bias [C] (used in float32)
    or None. Differentiable in x, weight and bias. Rows need unit stride of the
    last index (others are copied); any row pitch is read in place."""
    if x.ndim < 1:
        raise ValueError("x must have at least one dimension")
    c = x.shape[-1]
    if not 1 <= c <= MAX_WIDTH:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_WIDTH} values; got {c}")
    code_of("x", x)
    need_shape("weight", weight, (c,))
    need_shape("bias", bias, (c,))
    need_cuda("layer_norm", x, weight, bias)
    w, b = parameter(weight), parameter(bias)
    flat = rows(x if x.ndim == 2 else x.reshape(-1, c))
    if torch.compiler.is_compiling():
        y = torch.ops.spikegpt_b200.layer_norm(flat, w, b, float(eps))[0]
    else:
        guard = on_device(x)
        if guard is not None:
            with guard:
                return layer_norm(x, weight, bias, eps)
        y = _LayerNorm.apply(flat, w, b, float(eps)) if wants_grad(x, w, b) else _forward(flat, w, b, float(eps))[0]
    return y if x.ndim == 2 else y.view(x.shape)
