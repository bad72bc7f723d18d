"""GPU tests of ``layer_norm`` and ``q4_linear`` against their definitions in 64
bits: every type, widths from one on, odd widths and pitches, values far from
zero, gradients, group sizes, tokens, refusals."""

from __future__ import annotations

import pytest
import torch
from _mixertest import check, wide

import spikegpt_b200 as sg
from spikegpt_b200 import _capi

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


# --------------------------------------------------------------- layer norm


def _norm_ref(x, w, b, eps):
    d = x - x.mean(-1, keepdim=True)
    h = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return h * (1 if w is None else w) + (0 if b is None else b)


def _norm_case(shape, dtype, device, seed=0, shift=0.5):
    g = torch.Generator().manual_seed(seed + sum(shape))
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * 2 + shift).to(device, dtype).requires_grad_()
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(device).requires_grad_()
    b = (0.2 * torch.randn(c, generator=g)).to(device).requires_grad_()
    return x, w, b, torch.randn(shape, generator=g).to(device, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 33), (1, 512), (7, 130), (300, 96), (17, 1000), (4, 9, 1023),
                                   (33, 1024), (2, 2050), (65, 4096), (3, 8191), (9, 8192), (2, 16384), (2, 16383),
                                   (2000, 40)])  # fmt: skip
def test_layer_norm_and_gradients(cuda, shape, dtype):
    x, w, b, g = _norm_case(shape, dtype, cuda)
    y = sg.layer_norm(x, w, b)
    assert y.dtype == dtype and y.shape == x.shape
    refs = [wide(v) for v in (x, w, b)]
    ry = _norm_ref(*refs, 1e-5)
    check("y", y, ry)
    got = torch.autograd.grad(y, (x, w, b), g)
    want = torch.autograd.grad(ry, refs, g.double())
    # a width of one or two cancels to nothing: its gradient is measured against its terms, gy w rstd
    terms = g.double() * refs[1].detach() / torch.sqrt(refs[0].detach().var(-1, unbiased=False, keepdim=True) + 1e-5)
    check("gradient of x", got[0], want[0], scale_of=terms)
    check("gradient of weight", got[1], want[1])
    check("gradient of bias", got[2], want[2])
    with torch.no_grad():
        assert torch.equal(sg.layer_norm(x, w, b), y)


def test_layer_norm_without_parameters_and_single_gradients(cuda):
    x, w, b, g = _norm_case((6, 200), torch.float32, cuda, seed=3)
    refs = [wide(v) for v in (x, w, b)]
    for use_w, use_b in ((False, False), (True, False), (False, True)):
        ww, bb = (w if use_w else None), (b if use_b else None)
        y = sg.layer_norm(x, ww, bb)
        ry = _norm_ref(refs[0], refs[1] if use_w else None, refs[2] if use_b else None, 1e-5)
        check("y", y, ry)
        check("gradient of x", torch.autograd.grad(y, x, g)[0], torch.autograd.grad(ry, refs[0], g.double())[0])
    y = sg.layer_norm(x.detach(), w, None)
    check("gradient of weight alone", torch.autograd.grad(y, w, g)[0],
          torch.autograd.grad(_norm_ref(refs[0], refs[1], None, 1e-5), refs[1], g.double())[0])


def test_layer_norm_far_from_zero_and_constant_rows(cuda):
    """Statistics about the mean: rows at 300 with a spread of 1 lose 300 * 2^-24 of
    the spread at most; a constant row gives the bias."""
    x, w, b, _ = _norm_case((20, 777), torch.float32, cuda, seed=5)
    far = (x / 2 + 300.0).detach()
    ref = _norm_ref(far.double(), w.double(), b.double(), 1e-5)
    assert float((sg.layer_norm(far, w, b).double() - ref).abs().max()) <= 1e-4
    flat = torch.full((3, 777), 3.25, device=cuda)
    torch.testing.assert_close(sg.layer_norm(flat, w, b), b.expand(3, -1).float())


def test_layer_norm_row_pitches_and_empty(cuda):
    for dtype in (torch.float32, torch.bfloat16):
        holder = torch.randn(31, 205, device=cuda).to(dtype)
        for view in (holder[:, 3:203], holder[:, 4:204], holder[::2, :200], holder.t()[:200].t()):
            view = view.detach()
            w = torch.randn(view.shape[-1], device=cuda)
            want = sg.layer_norm(view.contiguous(), w)
            assert torch.equal(sg.layer_norm(view, w), want)
            a, c = view.clone().requires_grad_(), view.requires_grad_()
            ga = torch.autograd.grad(sg.layer_norm(a, w).float().sum(), a)[0]
            gc = torch.autograd.grad(sg.layer_norm(c, w).float().sum(), c)[0]
            assert torch.equal(ga, gc)
            view.requires_grad_(False)
    e = torch.zeros(0, 64, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    ge, gw = torch.autograd.grad(sg.layer_norm(e, w).sum(), (e, w))
    assert ge.shape == (0, 64) and (gw == 0).all()


def test_layer_norm_nan_stays_in_its_row(cuda):
    x, w, b, _ = _norm_case((9, 300), torch.bfloat16, cuda, seed=7)
    want = sg.layer_norm(x, w, b)
    bad = x.detach().clone()
    bad[4, 17] = float("nan")
    bad[6, 0] = float("inf")
    y = sg.layer_norm(bad, w, b)
    keep = [i for i in range(9) if i not in (4, 6)]
    assert torch.equal(y[keep], want[keep]) and y[4].isnan().all() and y[6].isnan().any()


def test_layer_norm_is_deterministic_and_checks_differences(cuda):
    x, w, b, g = _norm_case((500, 384), torch.float32, cuda, seed=9)
    runs = [torch.autograd.grad(sg.layer_norm(x, w, b), (x, w, b), g) for _ in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    for i, leaf in enumerate((x, w, b)):
        v = runs[0][i] / runs[0][i].abs().mean()
        sides = []
        for s in (1e-2, -1e-2):
            args = [(a + s * v if j == i else a).detach() for j, a in enumerate((x, w, b))]
            sides.append((sg.layer_norm(*args).double() * g.double()).sum())
        numeric, exact = float(sides[0] - sides[1]) / 2e-2, float((runs[0][i].double() * v.double()).sum())
        assert abs(numeric - exact) <= 5e-3 * abs(exact), i


def test_layer_norm_refusals(cuda):
    x = torch.zeros(4, 32, device=cuda)
    for args in ((x.double(),), (x.long(),), (x, torch.ones(31, device=cuda)), (x, None, torch.ones(33, device=cuda)),
                 (torch.zeros(2, 16385, device=cuda),), (torch.zeros(4, 0, device=cuda),), (x, torch.ones(32))):  # fmt: skip
        with pytest.raises(ValueError):
            sg.layer_norm(*args)
    with pytest.raises(NotImplementedError):
        sg.layer_norm(x.cpu())
    p = x.data_ptr()
    assert _capi.lib().layer_norm_backward(0, p, p, p, p, p, p, p, p, None, 0, 4, 32, 32, 32, None) == 2


# ------------------------------------------------------------ 4-bit weights


def _q4_case(m, k, n, g, dtype, device, zeros=True, seed=0):
    gen = torch.Generator().manual_seed(seed + m + 3 * k + 5 * n)
    w = torch.randn(n, k, generator=gen) / k**0.5
    packed, scales, zp = sg.quantize_q4(w.to(device), g, symmetric=not zeros)
    x = torch.randn(m, k, generator=gen).to(device, dtype)
    return x, packed, scales, zp


def _q4_ref(x, packed, scales, zp, k, g):
    return x.double() @ sg.dequantize_q4(packed, scales, zp, k, g).double().t()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,g", [(1, 32, 1, 32), (1, 64, 16, 64), (1, 768, 515, 64), (2, 100, 33, 32), (3, 1, 5, 32),
                                     (8, 513, 70, 128), (5, 1024, 129, 128), (6, 2047, 48, 64), (9, 320, 17, 96),
                                     (17, 256, 40, 256), (64, 512, 100, 64), (70, 130, 21, 32), (1, 8192, 64, 128),
                                     (4, 4096, 4097, 1024)])  # fmt: skip
def test_q4_linear(cuda, m, k, n, g, dtype):
    for zeros in (True, False):
        x, packed, scales, zp = _q4_case(m, k, n, g, dtype, cuda, zeros)
        ref = _q4_ref(x, packed, scales, zp, k, g)
        check("y", sg.q4_linear(x, packed, scales, zp, group_size=g), ref)
        bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(cuda)
        check("y with bias", sg.q4_linear(x, packed, scales, zp, bias, group_size=g), ref + bias.double())


def test_q4_what_lies_past_the_row_is_ignored(cuda):
    """Nibbles past K of any value; tokens at odd pitches, whose neighbours are NaN;
    leading dimensions; no tokens."""
    k, n, g = 75, 40, 64
    for dtype in TYPES:
        x, packed, scales, zp = _q4_case(3, k, n, g, dtype, cuda)
        want = sg.q4_linear(x, packed, scales, zp, group_size=g)
        full = packed.clone()
        full[:, (k + 1) // 2 :] = 0xF7
        full[:, k // 2] |= 0xF0  # k is odd: the high nibble of its last byte
        assert torch.equal(sg.q4_linear(x, full, scales, zp, group_size=g), want)
        holder = torch.full((3, k + 10), float("nan"), dtype=dtype, device=cuda)
        for at in (0, 1, 8):
            holder.fill_(float("nan"))
            holder[:, at : at + k] = x
            assert torch.equal(sg.q4_linear(holder[:, at : at + k], packed, scales, zp, group_size=g), want)
        assert torch.equal(sg.q4_linear(x.view(3, 1, k), packed, scales, zp, group_size=g), want.view(3, 1, n))
        assert torch.equal(sg.q4_linear(x[0], packed, scales, zp, group_size=g), want[0])
        assert sg.q4_linear(x[:0], packed, scales, zp, group_size=g).shape == (0, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 4, 5, 7, 9, 16, 19])
@pytest.mark.parametrize("k,n,g", [(256, 9504, 128), (130, 9511, 32), (388, 19000, 64)])
def test_q4_many_rows(cuda, m, k, n, g, dtype):
    """Rows enough to fill the GPU, where a warp takes twice as many; a token that is not
    finite touches no other."""
    x, packed, scales, zp = _q4_case(m, k, n, g, dtype, cuda, seed=m)
    ref = _q4_ref(x, packed, scales, zp, k, g)
    y = sg.q4_linear(x, packed, scales, zp, group_size=g)
    check("y", y, ref)
    x[m // 2, k // 3] = float("inf")
    spoilt = sg.q4_linear(x, packed, scales, zp, group_size=g)
    others = torch.arange(m, device=cuda) != m // 2
    assert torch.equal(spoilt[others], y[others])
    assert not torch.isfinite(spoilt[m // 2]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_q4_large_and_small_activations(cuda, dtype):
    """Tokens are independent: one at 1e4 beside one at 1e-3, and one with an infinity
    or a NaN, leave the others' values as they are."""
    x, packed, scales, zp = _q4_case(4, 512, 50, 64, dtype, cuda, seed=3)
    x[0] *= 1e4
    x[1] *= 1e-3
    ref = _q4_ref(x, packed, scales, zp, 512, 64)
    y = sg.q4_linear(x, packed, scales, zp, group_size=64)
    if dtype == torch.float16:
        ref[0] = ref[0].clamp(-65504, 65504)
        y[0] = y[0].clamp(-65504, 65504)
    for i in range(4):
        check(f"token {i}", y[i], ref[i])
    x[2, 5], x[3, 7] = float("nan"), float("inf")
    z = sg.q4_linear(x, packed, scales, zp, group_size=64)
    assert torch.equal(z[1], y[1]) and not torch.isfinite(z[2]).any()


def test_q4_refusals(cuda):
    x, packed, scales, zp = _q4_case(2, 64, 8, 64, torch.float32, cuda)
    for kw in (dict(group_size=48), dict(group_size=0), dict(group_size=32)):
        with pytest.raises(ValueError):
            sg.q4_linear(x, packed, scales, zp, **kw)
    for args in ((x[:, :30], packed, scales, zp), (x, packed.int(), scales, zp), (x, packed, scales.float(), zp),
                 (x, packed, scales[:4], zp), (x, packed, scales, zp.int()), (x.double(), packed, scales, zp),
                 (x, packed.t().contiguous().t(), scales, zp), (x, packed.cpu(), scales, zp),
                 (x, packed, scales, zp, torch.zeros(3, device=cuda))):  # fmt: skip
        with pytest.raises(ValueError):
            sg.q4_linear(*args)
    with pytest.raises(NotImplementedError):
        sg.q4_linear(x.clone().requires_grad_(), packed, scales, zp)
    with pytest.raises(NotImplementedError):
        sg.q4_linear(x.cpu(), packed, scales, zp)
    p = x.data_ptr()
    assert _capi.lib().q4_matvec(0, p, p, p, None, None, p, 1, 8, 64, 40, 64, None) == 1
