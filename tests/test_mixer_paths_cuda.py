"""GPU tests of the paths that only larger calls of the mixer operators take: a layer norm
whose CTAs walk several rows each, and scans split over time or not, at every layout of
the states, with the launches that show which."""

from __future__ import annotations

import pytest
import torch
from _mixertest import check, scan_inputs, scan_ref, wide

import spikegpt_b200 as sg
from spikegpt_b200 import _capi

pytestmark = pytest.mark.gpu

ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,c", [(12007, 96), (12007, 97), (4801, 515), (2501, 2048), (1501, 2050), (701, 8192),
                                    (701, 8191), (401, 16384), (401, 16383)])  # fmt: skip
def test_layer_norm_walks_rows(cuda, rows, c, dtype):
    """More rows than twice what all CTAs hold at a time (and no multiple of it), where words
    are aligned and where they go through shared memory. The sums over the rows may be off
    by the square root of as many float32 roundings, well inside the tests' allowance."""
    span = 32
    while span * 16 < c:
        span *= 2
    threads = max(256, span)
    at_a_time = 2 * torch.cuda.get_device_properties(cuda).multi_processor_count * 512 // threads * (threads // span)
    assert rows > 2 * at_a_time and rows % at_a_time
    g = torch.Generator().manual_seed(rows + c)
    x = (torch.randn(rows, c, generator=g) * 2 + 0.5).to(cuda, dtype).requires_grad_()
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(cuda).requires_grad_()
    b = (0.2 * torch.randn(c, generator=g)).to(cuda).requires_grad_()
    cot = torch.randn(rows, c, generator=g).to(cuda, dtype)
    refs = [wide(v) for v in (x, w, b)]
    off = refs[0] - refs[0].mean(-1, keepdim=True)
    ref = off / torch.sqrt((off * off).mean(-1, keepdim=True) + 1e-5) * refs[1] + refs[2]
    y = sg.layer_norm(x, w, b)
    check("y", y, ref)
    got = torch.autograd.grad(y, (x, w, b), cot)
    for name, a, r in zip(("x", "weight", "bias"), got, torch.autograd.grad(ref, refs, cot.double())):
        check(f"gradient of {name}", a, r)


@pytest.mark.parametrize("form", ["all", "no gate", "plain step"])
@pytest.mark.parametrize("b,t,c,n,split", [(1, 300, 70, 24, True), (2, 260, 40, 64, True), (1, 330, 66, 8, True),
                                           (1, 421, 130, 16, True), (100, 203, 130, 16, False), (100, 203, 66, 24, False),
                                           (50, 201, 96, 64, False), (150, 230, 65, 7, False)])  # fmt: skip
def test_scan_split_over_time_and_not(cuda, b, t, c, n, split, form):
    ins, h0, g = scan_inputs(b, t, c, n, torch.float32, cuda, seed=61)
    if form != "all":
        ins["z"] = None
    if form == "plain step":
        ins["dt"], ins["dt_bias"] = ins["dt"].abs() * 0.1, None
    softplus = form != "plain step"
    leaves = [None if ins[k] is None else ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    refs = [wide(v) for v in leaves]
    glast = torch.randn(h0.shape, generator=torch.Generator().manual_seed(1)).to(cuda)
    before = _capi.launch_counts()
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True, dt_softplus=softplus)
    has = [i for i, v in enumerate(leaves) if v is not None]
    got = torch.autograd.grad([out, last], [leaves[i] for i in has], [g, glast])
    after = _capi.launch_counts()
    for kernel in ("scan_summary_kernel", "scan_adjoint_kernel"):
        assert after[kernel] - before[kernel] == (1 if split else 0), kernel
    rout, rlast = scan_ref(*refs[:8], h0=refs[8], softplus=softplus)
    check("out", out, rout)
    check("last state", last, rlast)
    want = torch.autograd.grad([rout, rlast], [refs[i] for i in has], [g.double(), glast.double()])
    for i, a, r in zip(has, got, want):
        check(f"gradient of {(*ORDER, 'initial_state')[i]}", a, r)
