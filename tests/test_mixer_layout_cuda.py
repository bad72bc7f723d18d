"""GPU tests of the selective-mixer operators on parameters and weights that lie at
offsets of a flat buffer, where the words the kernels would like to move are not
aligned."""

from __future__ import annotations

import pytest
import torch
from _mixertest import check, scan_inputs, scan_ref, wide

import spikegpt_b200 as sg

pytestmark = pytest.mark.gpu

ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


def at_offset(t, offset=1):
    """A contiguous copy of t that starts `offset` elements into a buffer."""
    held = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)
    view = held[offset:].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,n", [(2, 37, 72, 16), (1, 19, 40, 8), (1, 300, 136, 24)])
@pytest.mark.parametrize("gated", [False, True])
def test_scan_with_unaligned_parameters_and_aligned_rows(cuda, gated, b, t, c, n, dtype):
    """Rows that move as 16-byte copies beside an A, D and dt_bias that do not: ragged last
    tiles in time and in channels, with z and without."""
    ins, _, g = scan_inputs(b, t, c, n, dtype, cuda, seed=41)
    if not gated:
        ins["z"] = None
    plain = [None if ins[k] is None else ins[k].detach().clone().requires_grad_() for k in ORDER]
    moved = [None if v is None else v.detach() for v in plain]
    for i in (2, 5, 7):
        moved[i] = at_offset(moved[i])
        assert moved[i].data_ptr() % 16 == 4 and moved[i].is_contiguous()
    moved = [None if v is None else v.requires_grad_() for v in moved]
    refs = [wide(v) for v in plain]
    out, ref = sg.selective_scan(*moved), scan_ref(*refs)[0]
    check("out", out, ref)
    assert torch.equal(out, sg.selective_scan(*plain))
    has = [i for i, v in enumerate(moved) if v is not None]
    got = torch.autograd.grad(out, [moved[i] for i in has], g)
    same = torch.autograd.grad(sg.selective_scan(*plain), [plain[i] for i in has], g)
    want = torch.autograd.grad(ref, [refs[i] for i in has], g.double())
    for i, a, p, r in zip(has, got, same, want):
        check(f"gradient of {ORDER[i]}", a, r)
        assert torch.equal(a, p), ORDER[i]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,g", [(1, 64, 33, 64), (5, 300, 70, 32), (20, 130, 9511, 128)])
def test_q4_weights_at_any_offset(cuda, m, k, n, g, dtype):
    """Packed weights, scales and zero points as views into flat buffers: the values of
    the same weights by themselves."""
    gen = torch.Generator().manual_seed(k)
    packed, scales, zeros = sg.quantize_q4((torch.randn(n, k, generator=gen) / k**0.5).to(cuda), g)
    x = torch.randn(m, k, generator=gen).to(cuda, dtype)
    want = sg.q4_linear(x, packed, scales, zeros, group_size=g)
    check("y", want, x.double() @ sg.dequantize_q4(packed, scales, zeros, k, g).double().t())
    for offset in (1, 2, 8, 16):
        moved = [at_offset(v, offset) for v in (packed, scales, zeros)]
        assert moved[0].data_ptr() % 16 == offset % 16
        assert torch.equal(sg.q4_linear(x, *moved, group_size=g), want)
