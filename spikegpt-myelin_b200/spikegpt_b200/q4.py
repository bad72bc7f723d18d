"""Projections with 4-bit weights for generation, on sm_100a.

At a few tokens a projection's time is its weights' bytes. ``quantize_q4`` stores a
weight [N, K] as 4-bit integers with one bfloat16 scale (and one zero point) for
each group of ``group_size`` inputs of a row: ``w ~ scale * (q - zero)``.
``q4_linear`` multiplies tokens by such a weight, decoding it in registers; the sums
are float32. No gradient: it serves generation.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._native import ops


def packed_pitch(in_features: int) -> int:
    """Bytes of one packed row."""
    return -(-in_features // 32) * 16


def quantize_q4(weight: Tensor, group_size: int = 64, *, symmetric: bool = False) -> tuple[Tensor, Tensor, Tensor | None]:
    """(packed uint8 [N, ceil(K/32)*16], scales bfloat16 [N, ceil(K/G)], zeros uint8
    of the scales' shape, or None when ``symmetric``: a zero point of 8 throughout).
    Weight k of a row is in byte k // 2, even k in the low nibble; the row is padded
    with zero weights to a multiple of 32. The integers are rounded against the
    scale as it is stored."""
    if weight.ndim != 2:
        raise ValueError(f"weight must have shape [N, K]; got {list(weight.shape)}")
    _check_group(group_size)
    n, k = weight.shape
    groups = -(-k // group_size)
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group_size - k)).view(n, groups, group_size)
    if symmetric:
        scale = (w.abs().amax(-1) / 7.0).to(torch.bfloat16)
        zero = torch.full((n, groups), 8.0, device=w.device)
    else:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((high - low) / 15.0).to(torch.bfloat16)
        zero = torch.where(scale > 0, torch.round(-low / scale.float()), torch.zeros_like(low)).clamp(0, 15)
    s = scale.float()[..., None]
    q = torch.where(s > 0, torch.round(w / s), torch.zeros_like(w)) + zero[..., None]
    q = q.clamp(0, 15).to(torch.uint8).view(n, groups * group_size)
    width = packed_pitch(k) * 2
    q = q[:, :width] if q.shape[1] >= width else torch.nn.functional.pad(q, (0, width - q.shape[1]))
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    return packed.contiguous(), scale.contiguous(), None if symmetric else zero.to(torch.uint8)


def dequantize_q4(packed: Tensor, scales: Tensor, zeros: Tensor | None, in_features: int, group_size: int) -> Tensor:
    """The float32 weight [N, K] that the packed form stands for."""
    _check_group(group_size)
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(1)[:, :in_features].float()
    group = torch.arange(in_features, device=packed.device) // group_size
    zero = 8.0 if zeros is None else zeros.float()[:, group]
    return (q - zero) * scales.float()[:, group]


def _check_group(group_size: int) -> None:
    if group_size < 32 or group_size % 32:
        raise ValueError(f"group_size must be a positive multiple of 32; got {group_size}")


def q4_linear(x: Tensor, packed: Tensor, scales: Tensor, zeros: Tensor | None = None, bias: Tensor | None = None, *,
              group_size: int = 64) -> Tensor:
    """``x @ W.T + bias`` for x [..., K] (CUDA, float32 / bfloat16 / float16) and the
    weight W [N, K] that ``quantize_q4`` packed with the same ``group_size``; in x's
    dtype. Made for up to 64 tokens a call (more run in turns that read the weight
    again). ``zeros`` may hold any byte (a row with one above 127 takes longer for
    bfloat16 and float32 tokens). A ``packed`` that is not 16-byte aligned (a view into a
    flat buffer) is copied at every call."""
    return ops.q4_linear(x, packed, scales, zeros, bias, group_size)
