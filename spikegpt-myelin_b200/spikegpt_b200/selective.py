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

from torch import Tensor

from ._native import ops

MAX_TAPS = 4
MAX_STATES = 64


def _kept_bytes(b: int, t: int, c: int, n: int) -> int:
    """Bytes of the states a differentiated scan keeps: every 8th step's, float32."""
    return b * ((t + 7) // 8) * c * n * 4


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
    y, state = ops.causal_conv(x, weight, bias, initial_state, lengths, silu, return_state)
    return (y, state) if return_state else y


def causal_conv_step_(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, *,
                      silu: bool = True) -> Tensor:
    """One token of ``causal_conv``: x [B, C], ``state`` [B, W-1, C] (contiguous, x's
    dtype) is moved on by x in place. No gradient."""
    return ops.causal_conv_step_(x, state, weight, bias, silu)


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
    out, state = ops.selective_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, lengths, dt_softplus, return_state)
    return (out, state) if return_state else out


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
    return ops.selective_scan_step_(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus)
