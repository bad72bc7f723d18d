"""64-bit reference forms of the selective-mixer operators, and the tolerances of
their tests.

float32 tensors: a result is a sum of products whose factors carry a few
roundings of 2^-24 each, and a state remembers at most some hundred steps, so
errors stay near 2^-24 times the square root of a few thousand roundings: 4e-6 of
the tensor's largest value; TOL_F32 allows 2e-5. 16-bit tensors: the float32
result rounded once, half an ulp: 2^-9 (bfloat16) or 2^-12 (float16) of the value
itself, with the float32 allowance beside it; the tests allow a whole ulp.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

TOL_F32 = 2e-5
ULP = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
F16_SMALLEST = 2.0**-24  # below this a float16 is a subnormal's rounding


def check(name, got, ref, *, scale_of=None):
    """|got - ref| <= ulp |ref| + TOL_F32 max|ref|, element by element, NaNs and all."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if got.numel() == 0:
        return
    g, r = got.detach().double(), ref.detach().double()
    assert torch.isfinite(g).all(), f"{name} is not finite everywhere"
    scale = float((r if scale_of is None else scale_of).abs().max())
    room = ULP[got.dtype] * r.abs() + TOL_F32 * scale + (F16_SMALLEST if got.dtype == torch.float16 else 1e-30)
    worst = float(((g - r).abs() / room).max())
    assert worst <= 1.0, f"{name}: {worst:.2f} times the tolerance"


def conv_ref(x, weight, bias, window=None, silu=True, lengths=None):
    """(y, new window) in the inputs' (64-bit) type, differentiable."""
    b, t, c = x.shape
    w = weight.shape[1]
    if lengths is not None:  # what lies past the length is not looked at
        keep = (torch.arange(t, device=x.device)[None] < lengths[:, None].clamp(0, t))[..., None]
        x = torch.where(keep, x, torch.zeros_like(x))
    full = torch.cat([x.new_zeros(b, w - 1, c) if window is None else window, x], 1)
    u = sum(weight[:, j] * full[:, j : j + t] for j in range(w))
    if bias is not None:
        u = u + bias
    y = u * torch.sigmoid(u) if silu else u
    if lengths is None:
        return y, full[:, t:]
    y = torch.where(keep, y, torch.zeros_like(y))
    ends = [int(n) for n in lengths.clamp(0, t)]
    return y, torch.stack([full[i, n : n + w - 1] for i, n in enumerate(ends)])


def scan_ref(x, dt, A, B, C, D=None, z=None, dt_bias=None, h0=None, softplus=True, lengths=None):
    """(out, last state) step by step, differentiable."""
    b, t, c = x.shape
    raw = dt if dt_bias is None else dt + dt_bias
    delta = F.softplus(raw, threshold=40.0) if softplus else raw
    h = x.new_zeros(b, c, A.shape[1]) if h0 is None else h0
    outs = []
    for i in range(t):
        d, xi, Bi, Ci = delta[:, i], x[:, i], B[:, i], C[:, i]
        zi = None if z is None else z[:, i]
        if lengths is not None:
            live = (i < lengths)[:, None]
            d, xi, Bi, Ci = (torch.where(live, v, torch.zeros_like(v)) for v in (d, xi, Bi, Ci))
            zi = None if zi is None else torch.where(live, zi, torch.zeros_like(zi))
        h = torch.exp(d[..., None] * A) * h + (d * xi)[..., None] * Bi[:, None]
        y = (h * Ci[:, None]).sum(-1)
        if D is not None:
            y = y + D * xi
        if zi is not None:
            y = y * zi * torch.sigmoid(zi)
        if lengths is not None:
            y = torch.where(live, y, torch.zeros_like(y))
        outs.append(y)
    return (torch.stack(outs, 1) if outs else x.new_zeros(x.shape)), h


def wide(t):
    """A 64-bit copy that requires grad (None stays None)."""
    return None if t is None else t.detach().double().requires_grad_()


def scan_inputs(b, t, c, n, dtype, device, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed + 131 * b + 17 * t + c + n)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g) * scale

    x, dt, z = normal(b, t, c), normal(b, t, c, scale=0.5), normal(b, t, c)
    B, C = normal(b, t, n), normal(b, t, n)
    A = -torch.arange(1, n + 1).float() * torch.exp(0.1 * normal(c, n))
    D, bias = 1 + 0.1 * normal(c), -3.0 + normal(c)
    io = {k: v.to(device=device, dtype=dtype) for k, v in {"x": x, "dt": dt, "B": B, "C": C, "z": z}.items()}
    par = {k: v.to(device) for k, v in {"A": A, "D": D, "dt_bias": bias}.items()}
    return {**io, **par}, normal(b, c, n, scale=0.5).to(device), normal(b, t, c).to(device=device, dtype=dtype)
