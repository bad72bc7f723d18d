"""GPU tests of ``q4_linear`` with zero points of any byte."""

from __future__ import annotations

import pytest
import torch
from _mixertest import check

import spikegpt_b200 as sg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,g", [(1, 64, 33, 64), (3, 301, 70, 32), (9, 256, 9511, 128), (20, 130, 48, 64),
                                     (6, 1024, 40, 1024), (5, 2048, 9500, 64)])  # fmt: skip
def test_zero_points_of_any_byte(cuda, m, k, n, g, dtype):
    """Every value of a byte, from rows that have none above 127 to rows that have only such;
    the rows without one keep their values to the bit, whatever their neighbours hold."""
    gen = torch.Generator().manual_seed(m + k + n)
    packed, scales, plain = sg.quantize_q4((torch.randn(n, k, generator=gen) / k**0.5).to(cuda), g)
    x = torch.randn(m, k, generator=gen).to(cuda, dtype)
    bias = torch.randn(n, generator=gen).to(cuda)
    groups = scales.shape[1]
    any_byte = torch.randint(0, 256, (n, groups), generator=gen, dtype=torch.uint8).to(cuda)
    kind = torch.arange(n, device=cuda) % 4
    zeros = plain.clone()
    zeros[kind == 1] = any_byte[kind == 1]
    zeros[kind == 2] = any_byte[kind == 2] | 128
    zeros[kind == 3, groups // 2] = 129
    ref = x.double() @ sg.dequantize_q4(packed, scales, zeros, k, g).double().t()
    y = sg.q4_linear(x, packed, scales, zeros, group_size=g)
    check("y", y, ref)
    check("y with bias", sg.q4_linear(x, packed, scales, zeros, bias, group_size=g), ref + bias.double())
    assert torch.equal(y[:, kind == 0], sg.q4_linear(x, packed, scales, plain, group_size=g)[:, kind == 0])
    x[m // 2, k // 3] = float("nan")
    spoilt = sg.q4_linear(x, packed, scales, zeros, group_size=g)
    assert spoilt[m // 2].isnan().all()
    others = torch.arange(m, device=cuda) != m // 2
    assert torch.equal(spoilt[others], y[others])
