"""Selective state-space scan and its short causal convolution, on sm_100a.

A second time mixing next to WKV and RWKV-7 (the reference has no counterpart):
each channel c keeps N states whose decay and input depend on the token,

    d_t = softplus(dt_t + dt_bias)
    h_t = exp(d_t A) * h_{t-1} + d_t x_t B_t          (A [C, N]; B_t, C_t [N])
    y_t = (C_t . h_t + D x_t) * silu(z_t)

on inputs that a causal convolution of each channel with its own W <= 4 taps has
gone over. ``causal_conv`` and ``selective_scan`` take sequences [B, T, C], for
training (every input and parameter has a gradient) and for prompts (they start
from and return the states, and take right-padded batches by ``lengths``);
``causal_conv_step_`` and ``selective_scan_step_`` take one token [B, C] and move
the states on in place. float32, bfloat16 and float16 tensors; the state, the
parameters and every sum are float32.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _capi
from ._mixer import (
    code_of,
    lengths_of,
    need_cuda,
    need_dtype,
    need_shape,
    no_grad_only,
    on_device,
    parameter,
    ptr,
    rows,
    stream,
    wants_grad,
    workspace,
)

MAX_TAPS = 4
MAX_STATES = 64


# ------------------------------------------------------- causal convolution


def _conv_forward(x: Tensor, weight: Tensor, bias: Tensor | None, window: Tensor | None, lengths: Tensor | None,
                  silu: bool, want_window: bool) -> tuple[Tensor, Tensor]:
    b, t, c = x.shape
    w = weight.shape[1]
    y = torch.empty((b, t, c), dtype=x.dtype, device=x.device)
    new = torch.empty((b, w - 1, c) if want_window else 0, dtype=x.dtype, device=x.device)
    _capi.check(
        _capi.lib().causal_conv_forward(code_of("x", x), x.data_ptr(), weight.data_ptr(), ptr(bias), ptr(window),
                                        ptr(lengths), y.data_ptr(), new.data_ptr() if want_window else None, b, t, c,
                                        w, x.stride(0), x.stride(1), silu, stream(x)),
        "causal_conv_forward",
    )
    return y, new


def _conv_backward(g: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None, window: Tensor | None,
                   lengths: Tensor | None, silu: bool, want_window: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    b, t, c = x.shape
    w = weight.shape[1]
    lib = _capi.lib()
    gx = torch.empty((b, t, c), dtype=x.dtype, device=x.device)
    gw = torch.empty((c, w), dtype=torch.float32, device=x.device)
    gb = torch.empty(c if bias is not None else 0, dtype=torch.float32, device=x.device)
    gwin = torch.empty((b, w - 1, c) if want_window else 0, dtype=x.dtype, device=x.device)
    nws = lib.causal_conv_workspace_size(b, t, c, w)
    ws = workspace(nws, x)
    _capi.check(
        lib.causal_conv_backward(code_of("x", x), g.data_ptr(), x.data_ptr(), weight.data_ptr(), ptr(bias),
                                 ptr(window), ptr(lengths), gx.data_ptr(), gw.data_ptr(),
                                 gb.data_ptr() if bias is not None else None,
                                 gwin.data_ptr() if want_window else None, ptr(ws), nws, b, t, c, w, g.stride(0),
                                 g.stride(1), x.stride(0), x.stride(1), silu, stream(x)),
        "causal_conv_backward",
    )
    return gx, gw, gb, gwin


@torch.library.custom_op("spikegpt_b200::causal_conv", mutates_args=(), device_types="cuda")
def _conv_op(x: Tensor, weight: Tensor, bias: Tensor | None, window: Tensor | None, lengths: Tensor | None,
             silu: bool, want_window: bool) -> tuple[Tensor, Tensor]:
    with on_device(x) or nullcontext():
        return _conv_forward(rows(x), weight, bias, window, lengths, silu, want_window)


@_conv_op.register_fake
def _(x, weight, bias, window, lengths, silu, want_window):
    b, _, c = x.shape
    return x.new_empty(x.shape), x.new_empty((b, weight.shape[1] - 1, c) if want_window else (0,))


@torch.library.custom_op("spikegpt_b200::causal_conv_backward", mutates_args=(), device_types="cuda")
def _conv_op_backward(g: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None, window: Tensor | None,
                      lengths: Tensor | None, silu: bool,
                      want_window: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    with on_device(x) or nullcontext():
        return _conv_backward(rows(g), rows(x), weight, bias, window, lengths, silu, want_window)


@_conv_op_backward.register_fake
def _(g, x, weight, bias, window, lengths, silu, want_window):
    b, _, c = x.shape
    return (x.new_empty(x.shape), torch.empty_like(weight),
            x.new_empty(c if bias is not None else 0, dtype=torch.float32),
            x.new_empty((b, weight.shape[1] - 1, c) if want_window else (0,)))


def _conv_setup(ctx, inputs, output):
    x, weight, bias, window, lengths, silu, _want = inputs
    ctx.save_for_backward(x, weight, bias, window, lengths)
    ctx.silu = silu
    ctx.mark_non_differentiable(output[1])


def _conv_op_grad(ctx, g, _gwindow):
    x, weight, bias, window, lengths = ctx.saved_tensors
    gx, gw, gb, gwin = torch.ops.spikegpt_b200.causal_conv_backward(g.to(x.dtype), x, weight, bias, window, lengths,
                                                                    ctx.silu, window is not None)
    return gx, gw, gb if bias is not None else None, gwin if window is not None else None, None, None, None


_conv_op.register_autograd(_conv_op_grad, setup_context=_conv_setup)


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, window, lengths, silu):
        ctx.save_for_backward(x, weight, bias, window, lengths)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, window, lengths, silu, False)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, window, lengths = ctx.saved_tensors
        with on_device(x) or nullcontext():
            gx, gw, gb, gwin = _conv_backward(rows(g), x, weight, bias, window, lengths, ctx.silu,
                                              ctx.needs_input_grad[3])
        return gx, gw, gb if bias is not None else None, gwin if ctx.needs_input_grad[3] else None, None, None


def _last_rows(x: Tensor, window: Tensor | None, lengths: Tensor | None, w: int) -> Tensor:
    """The new window in torch operations (a copy of rows, with autograd's gradient)."""
    b, t, c = x.shape
    full = torch.cat([x.new_zeros(b, w - 1, c) if window is None else window, x], 1)
    if lengths is None:
        return full[:, t:].contiguous()
    at = lengths.long().clamp(0, t)[:, None] + torch.arange(w - 1, device=x.device)
    return torch.gather(full, 1, at[..., None].expand(-1, -1, c))


def _conv_weight(weight: Tensor, c: int) -> int:
    if weight.ndim != 2 or weight.shape[0] != c or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"weight must have shape [C={c}, W] with W from 1 to {MAX_TAPS}; got {list(weight.shape)}")
    return weight.shape[1]


def causal_conv(
    x: Tensor,
    weight: Tensor,
    bias: Tensor | None = None,
    *,
    silu: bool = True,
    initial_state: Tensor | None = None,
    lengths: Tensor | None = None,
    return_state: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """``silu(bias + sum_j weight[:, j] x[t - W + 1 + j])`` for x [B, T, C] (CUDA) and
    weight [C, W], W <= 4; without ``silu``, the sum itself. ``initial_state``
    [B, W-1, C] holds the rows before the first (default zeros); ``return_state``
    adds the last W - 1 rows to the result, the next call's initial state. With
    ``lengths`` [B], what lies past a sequence's length is not read, gives zeros and
    has no gradient. Differentiable in x, weight, bias and initial_state."""
    if x.ndim != 3:
        raise ValueError(f"x must have shape [B, T, C]; got {list(x.shape)}")
    b, _, c = x.shape
    w = _conv_weight(weight, c)
    code_of("x", x)
    need_shape("bias", bias, (c,))
    need_shape("initial_state", initial_state, (b, w - 1, c))
    need_dtype("initial_state", initial_state, x.dtype, "x")
    need_cuda("causal_conv", x, weight, bias, initial_state, lengths)
    wt, bi, lens = parameter(weight), parameter(bias), lengths_of(lengths, b)
    window = None if initial_state is None else initial_state.contiguous()
    x = rows(x)
    if torch.compiler.is_compiling():
        y, _ = torch.ops.spikegpt_b200.causal_conv(x, wt, bi, window, lens, silu, False)
        return (y, _last_rows(x, window, lens, w)) if return_state else y
    guard = on_device(x)
    if guard is not None:
        with guard:
            return causal_conv(x, weight, bias, silu=silu, initial_state=initial_state, lengths=lengths,
                               return_state=return_state)
    if wants_grad(x, wt, bi, window):
        y = _Conv.apply(x, wt, bi, window, lens, silu)
        return (y, _last_rows(x, window, lens, w)) if return_state else y
    y, new = _conv_forward(x, wt, bi, window, lens, silu, return_state)
    return (y, new) if return_state else y


def _conv_step(x: Tensor, window: Tensor, weight: Tensor, bias: Tensor | None, silu: bool) -> Tensor:
    b, c = x.shape
    y = torch.empty((b, c), dtype=x.dtype, device=x.device)
    _capi.check(
        _capi.lib().causal_conv_step(code_of("x", x), x.data_ptr(), weight.data_ptr(), ptr(bias), window.data_ptr(),
                                     y.data_ptr(), b, c, weight.shape[1], x.stride(0), silu, stream(x)),
        "causal_conv_step",
    )
    return y


@torch.library.custom_op("spikegpt_b200::causal_conv_step_", mutates_args=("window",), device_types="cuda")
def _conv_step_op(x: Tensor, window: Tensor, weight: Tensor, bias: Tensor | None, silu: bool) -> Tensor:
    with on_device(x) or nullcontext():
        return _conv_step(rows(x), window, weight, bias, silu)


@_conv_step_op.register_fake
def _(x, window, weight, bias, silu):
    return x.new_empty(x.shape)


def causal_conv_step_(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, *,
                      silu: bool = True) -> Tensor:
    """One token of ``causal_conv``: x [B, C], ``state`` [B, W-1, C] (contiguous, x's
    dtype) is moved on by x in place. No gradient."""
    if x.ndim != 2:
        raise ValueError(f"x must have shape [B, C]; got {list(x.shape)}")
    b, c = x.shape
    w = _conv_weight(weight, c)
    code_of("x", x)
    need_shape("state", state, (b, w - 1, c))
    need_dtype("state", state, x.dtype, "x")
    need_shape("bias", bias, (c,))
    need_cuda("causal_conv_step_", x, state, weight, bias)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous")
    no_grad_only("causal_conv_step_", x, state, weight, bias)
    wt, bi, x = parameter(weight), parameter(bias), rows(x)
    if torch.compiler.is_compiling():
        return torch.ops.spikegpt_b200.causal_conv_step_(x, state, wt, bi, silu)
    guard = on_device(x)
    if guard is not None:
        with guard:
            return _conv_step(x, state, wt, bi, silu)
    return _conv_step(x, state, wt, bi, silu)


# --------------------------------------------------------------------- scan


def _scan_forward(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None, z: Tensor | None,
                  dt_bias: Tensor | None, h0: Tensor | None, lengths: Tensor | None, softplus: bool, want_last: bool,
                  want_kept: bool) -> tuple[Tensor, Tensor, Tensor]:
    b, t, c = x.shape
    n = A.shape[1]
    code = code_of("x", x)
    lib = _capi.lib()
    out = torch.empty((b, t, c), dtype=x.dtype, device=x.device)
    last = torch.empty((b, c, n) if want_last else 0, dtype=torch.float32, device=x.device)
    nkept = lib.selective_scan_state_size(b, t, c, n) if want_kept else 0
    kept = torch.empty(nkept, dtype=torch.uint8, device=x.device)
    nws = lib.selective_scan_forward_workspace_size(code, b, t, c, n)
    ws = workspace(nws, x)
    zs = (0, 0) if z is None else (z.stride(0), z.stride(1))
    _capi.check(
        lib.selective_scan_forward(code, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), ptr(D),
                                   ptr(z), ptr(dt_bias), ptr(h0), ptr(lengths), out.data_ptr(),
                                   last.data_ptr() if want_last else None, kept.data_ptr() if want_kept else None,
                                   nkept, ptr(ws), nws, b, t, c, n, x.stride(0), x.stride(1), dt.stride(0),
                                   dt.stride(1), B.stride(0), B.stride(1), C.stride(0), C.stride(1), *zs, softplus,
                                   stream(x)),
        "selective_scan_forward",
    )
    return out, last, kept


def _scan_backward(g: Tensor, x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None,
                   z: Tensor | None, dt_bias: Tensor | None, lengths: Tensor | None, kept: Tensor,
                   glast: Tensor | None, softplus: bool, want_h0: bool) -> tuple[Tensor, ...]:
    """Gradients of x, dt, A, B, C, D, z, dt_bias and the initial state; empty
    tensors for the inputs that are None (and for a state that is not asked for)."""
    b, t, c = x.shape
    n = A.shape[1]
    code = code_of("x", x)
    lib = _capi.lib()
    dev, f32 = x.device, torch.float32
    gx, gdt = torch.empty((2, b, t, c), dtype=x.dtype, device=dev).unbind(0)
    gB, gC = torch.empty((2, b, t, n), dtype=x.dtype, device=dev).unbind(0)
    gA = torch.empty((c, n), dtype=f32, device=dev)
    gD = torch.empty(c if D is not None else 0, dtype=f32, device=dev)
    gz = torch.empty((b, t, c) if z is not None else 0, dtype=x.dtype, device=dev)
    gbias = torch.empty(c if dt_bias is not None else 0, dtype=f32, device=dev)
    gh0 = torch.empty((b, c, n) if want_h0 else 0, dtype=f32, device=dev)
    nws = lib.selective_scan_backward_workspace_size(code, b, t, c, n)
    ws = workspace(nws, x)
    zs = (0, 0) if z is None else (z.stride(0), z.stride(1))
    _capi.check(
        lib.selective_scan_backward(code, g.data_ptr(), x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
                                    C.data_ptr(), ptr(D), ptr(z), ptr(dt_bias), kept.data_ptr(), ptr(lengths),
                                    ptr(glast), gx.data_ptr(), gdt.data_ptr(), gA.data_ptr(), gB.data_ptr(),
                                    gC.data_ptr(), gD.data_ptr() if D is not None else None,
                                    gz.data_ptr() if z is not None else None,
                                    gbias.data_ptr() if dt_bias is not None else None,
                                    gh0.data_ptr() if want_h0 else None, ptr(ws), nws, b, t, c, n, g.stride(0),
                                    g.stride(1), x.stride(0), x.stride(1), dt.stride(0), dt.stride(1), B.stride(0),
                                    B.stride(1), C.stride(0), C.stride(1), *zs, softplus, stream(x)),
        "selective_scan_backward",
    )
    return gx, gdt, gA, gB, gC, gD, gz, gbias, gh0


@torch.library.custom_op("spikegpt_b200::selective_scan", mutates_args=(), device_types="cuda")
def _scan_op(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None, z: Tensor | None,
             dt_bias: Tensor | None, h0: Tensor | None, lengths: Tensor | None, softplus: bool, want_last: bool,
             want_kept: bool) -> tuple[Tensor, Tensor, Tensor]:
    with on_device(x) or nullcontext():
        return _scan_forward(rows(x), rows(dt), A, rows(B), rows(C), D, rows(z), dt_bias, h0, lengths, softplus,
                             want_last, want_kept)


def _kept_bytes(b, t, c, n):
    return b * ((t + 7) // 8) * c * n * 4


@_scan_op.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want_last, want_kept):
    b, t, c = x.shape
    n = A.shape[1]
    return (x.new_empty(x.shape), x.new_empty((b, c, n) if want_last else (0,), dtype=torch.float32),
            x.new_empty(_kept_bytes(b, t, c, n) if want_kept else 0, dtype=torch.uint8))


@torch.library.custom_op("spikegpt_b200::selective_scan_backward", mutates_args=(), device_types="cuda")
def _scan_op_backward(g: Tensor, x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None,
                      z: Tensor | None, dt_bias: Tensor | None, lengths: Tensor | None, kept: Tensor,
                      glast: Tensor | None, softplus: bool, want_h0: bool) -> list[Tensor]:
    with on_device(x) or nullcontext():
        got = _scan_backward(rows(g), rows(x), rows(dt), A, rows(B), rows(C), D, rows(z), dt_bias, lengths, kept,
                             None if glast is None else glast.contiguous(), softplus, want_h0)
    gx, gdt, gA, gB, gC, *rest = got
    return [gx, gdt.clone(), gA, gB, gC.clone(), *rest]  # a custom op's outputs share no memory


@_scan_op_backward.register_fake
def _(g, x, dt, A, B, C, D, z, dt_bias, lengths, kept, glast, softplus, want_h0):
    b, t, c = x.shape
    n, f32 = A.shape[1], torch.float32
    return [x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((c, n), dtype=f32), x.new_empty((b, t, n)),
            x.new_empty((b, t, n)), x.new_empty(c if D is not None else 0, dtype=f32),
            x.new_empty(x.shape if z is not None else (0,)), x.new_empty(c if dt_bias is not None else 0, dtype=f32),
            x.new_empty((b, c, n) if want_h0 else (0,), dtype=f32)]


def _scan_setup(ctx, inputs, output):
    x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want_last, _want_kept = inputs
    ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, output[2])
    ctx.softplus, ctx.want_last, ctx.has_h0 = softplus, want_last, h0 is not None
    ctx.mark_non_differentiable(output[2])


def _scan_op_grad(ctx, g, glast, _gkept):
    x, dt, A, B, C, D, z, dt_bias, lengths, kept = ctx.saved_tensors
    if g is None:
        g = torch.zeros_like(x)
    got = torch.ops.spikegpt_b200.selective_scan_backward(
        g.to(x.dtype), x, dt, A, B, C, D, z, dt_bias, lengths, kept, glast if ctx.want_last else None, ctx.softplus,
        ctx.has_h0)
    has = (True, True, True, True, True, D is not None, z is not None, dt_bias is not None, ctx.has_h0)
    return (*(v if h else None for v, h in zip(got, has)), None, None, None, None)


_scan_op.register_autograd(_scan_op_grad, setup_context=_scan_setup)


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want_last):
        out, last, kept = _scan_forward(x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want_last, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, kept)
        ctx.softplus, ctx.want_last = softplus, want_last
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g, glast):
        x, dt, A, B, C, D, z, dt_bias, lengths, kept = ctx.saved_tensors
        if g is None:
            g = torch.zeros_like(x)
        want_h0 = ctx.needs_input_grad[8]
        with on_device(x) or nullcontext():
            got = _scan_backward(rows(g), x, dt, A, B, C, D, z, dt_bias, lengths, kept,
                                 glast.contiguous() if ctx.want_last and glast is not None else None, ctx.softplus,
                                 want_h0)
        has = (True, True, True, True, True, D is not None, z is not None, dt_bias is not None, want_h0)
        return (*(v if h else None for v, h in zip(got, has)), None, None, None)


def _scan_parameters(A: Tensor, D: Tensor | None, dt_bias: Tensor | None, c: int) -> int:
    if A.ndim != 2 or A.shape[0] != c or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must have shape [C={c}, N] with N from 1 to {MAX_STATES}; got {list(A.shape)}")
    need_shape("D", D, (c,))
    need_shape("dt_bias", dt_bias, (c,))
    return A.shape[1]


def selective_scan(
    x: Tensor,
    dt: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    dt_bias: Tensor | None = None,
    *,
    dt_softplus: bool = True,
    initial_state: Tensor | None = None,
    lengths: Tensor | None = None,
    return_state: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """The selective scan of x, dt, z [B, T, C] with B, C [B, T, N] (CUDA, one dtype;
    any row pitch is read in place, so slices of a wider projection need no copy)
    and the float32 parameters A [C, N], D [C], dt_bias [C], N <= 64:

        d = softplus(dt + dt_bias)  (``dt_softplus=False``: dt + dt_bias)
        h = exp(d A) * h + d x B;  out = (C . h + D x) * silu(z)

    D, z and dt_bias may be None. ``initial_state`` [B, C, N] is float32 (default
    zeros); ``return_state`` adds the last state to the result. With ``lengths`` [B],
    what lies past a sequence's length is not read, gives zeros, and leaves the
    state as it is. Differentiable in every tensor but lengths; the backward keeps
    the state of every 8th step (float32, N / 2 bytes for each element of x)."""
    if x.ndim != 3:
        raise ValueError(f"x must have shape [B, T, C]; got {list(x.shape)}")
    b, t, c = x.shape
    n = _scan_parameters(A, D, dt_bias, c)
    code_of("x", x)
    need_shape("dt", dt, (b, t, c))
    need_shape("z", z, (b, t, c))
    need_shape("B", B, (b, t, n))
    need_shape("C", C, (b, t, n))
    for name, v in (("dt", dt), ("B", B), ("C", C), ("z", z)):
        need_dtype(name, v, x.dtype, "x")
    need_shape("initial_state", initial_state, (b, c, n))
    if initial_state is not None and initial_state.dtype != torch.float32:
        raise ValueError(f"initial_state must be float32; got {initial_state.dtype}")
    need_cuda("selective_scan", x, dt, A, B, C, D, z, dt_bias, initial_state, lengths)
    At, Dt, bt, lens = parameter(A), parameter(D), parameter(dt_bias), lengths_of(lengths, b)
    h0 = None if initial_state is None else initial_state.contiguous()
    x, dt, B, C, z = rows(x), rows(dt), rows(B), rows(C), rows(z)
    grad = wants_grad(x, dt, At, B, C, Dt, z, bt, h0)
    if torch.compiler.is_compiling():
        out, last, _ = torch.ops.spikegpt_b200.selective_scan(x, dt, At, B, C, Dt, z, bt, h0, lens, dt_softplus,
                                                              return_state, grad)
        return (out, last) if return_state else out
    guard = on_device(x)
    if guard is not None:
        with guard:
            return selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus=dt_softplus,
                                  initial_state=initial_state, lengths=lengths, return_state=return_state)
    if grad:
        out, last = _Scan.apply(x, dt, At, B, C, Dt, z, bt, h0, lens, dt_softplus, return_state)
    else:
        out, last, _ = _scan_forward(x, dt, At, B, C, Dt, z, bt, h0, lens, dt_softplus, return_state, False)
    return (out, last) if return_state else out


def _scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None,
               z: Tensor | None, dt_bias: Tensor | None, softplus: bool) -> Tensor:
    b, c = x.shape
    out = torch.empty((b, c), dtype=x.dtype, device=x.device)
    _capi.check(
        _capi.lib().selective_scan_step(code_of("x", x), x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
                                        C.data_ptr(), state.data_ptr(), ptr(D), ptr(z), ptr(dt_bias), out.data_ptr(),
                                        b, c, A.shape[1], x.stride(0), dt.stride(0), B.stride(0), C.stride(0),
                                        0 if z is None else z.stride(0), softplus, stream(x)),
        "selective_scan_step",
    )
    return out


@torch.library.custom_op("spikegpt_b200::selective_scan_step_", mutates_args=("state",), device_types="cuda")
def _scan_step_op(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None,
                  z: Tensor | None, dt_bias: Tensor | None, softplus: bool) -> Tensor:
    with on_device(x) or nullcontext():
        return _scan_step(rows(x), rows(dt), A, rows(B), rows(C), state, D, rows(z), dt_bias, softplus)


@_scan_step_op.register_fake
def _(x, dt, A, B, C, state, D, z, dt_bias, softplus):
    return x.new_empty(x.shape)


def selective_scan_step_(
    x: Tensor,
    dt: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    state: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    dt_bias: Tensor | None = None,
    *,
    dt_softplus: bool = True,
) -> Tensor:
    """One token of ``selective_scan``: x, dt, z [B, C] and B, C [B, N]; ``state``
    [B, C, N] (float32, contiguous) is moved on in place. No gradient."""
    if x.ndim != 2:
        raise ValueError(f"x must have shape [B, C]; got {list(x.shape)}")
    b, c = x.shape
    n = _scan_parameters(A, D, dt_bias, c)
    code_of("x", x)
    if dt.shape != x.shape or (z is not None and z.shape != x.shape) or B.shape != (b, n) or C.shape != (b, n):
        raise ValueError(f"dt and z must have shape {[b, c]} and B and C {[b, n]}; got {list(dt.shape)}, "
                         f"{None if z is None else list(z.shape)}, {list(B.shape)} and {list(C.shape)}")
    dtype = x.dtype
    if dt.dtype != dtype or B.dtype != dtype or C.dtype != dtype or (z is not None and z.dtype != dtype):
        raise ValueError(f"dt, B, C and z must have the dtype of x ({dtype})")
    if state.shape != (b, c, n) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 {[b, c, n]}; got {state.dtype} {list(state.shape)}")
    need_cuda("selective_scan_step_", x, dt, A, B, C, state, D, z, dt_bias)
    no_grad_only("selective_scan_step_", x, dt, A, B, C, state, D, z, dt_bias)
    At, Dt, bt = parameter(A), parameter(D), parameter(dt_bias)
    x, dt, B, C, z = rows(x), rows(dt), rows(B), rows(C), rows(z)
    if torch.compiler.is_compiling():
        return torch.ops.spikegpt_b200.selective_scan_step_(x, dt, At, B, C, state, Dt, z, bt, dt_softplus)
    guard = on_device(x)
    if guard is not None:
        with guard:
            return _scan_step(x, dt, At, B, C, state, Dt, z, bt, dt_softplus)
    return _scan_step(x, dt, At, B, C, state, Dt, z, bt, dt_softplus)
