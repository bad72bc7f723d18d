"""GPU tests of the selective scan and the short causal convolution against their
definitions in 64 bits (``_mixertest``): every type, lengths from zero on, odd
channel counts and state sizes, strided inputs, right-padded batches with NaN in
the padding, carried states, gradients (against the formula's and against
differences), the single-token steps against the sequence form, and refusals."""

from __future__ import annotations

import pytest
import torch
from _mixertest import check, conv_ref, scan_inputs, scan_ref, wide

import spikegpt_b200 as sg
from spikegpt_b200 import _capi

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


def _grads(outs, cots, leaves):
    return torch.autograd.grad(outs, leaves, cots, allow_unused=True)


# --------------------------------------------------------------------- scan


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "b,t,c,n",
    [(1, 1, 1, 1), (2, 17, 33, 16), (1, 16, 64, 16), (3, 31, 130, 8), (2, 65, 40, 5), (1, 150, 67, 16), (2, 33, 70, 24),
     (1, 40, 36, 64), (5, 2, 260, 13)],
)  # fmt: skip
def test_scan_outputs_and_gradients(cuda, b, t, c, n, dtype):
    ins, h0, g = scan_inputs(b, t, c, n, dtype, cuda)
    glast = torch.randn(h0.shape, generator=torch.Generator().manual_seed(1)).to(cuda)
    leaves = [ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True)
    refs = [wide(v) for v in leaves]
    rout, rlast = scan_ref(*refs[:8], h0=refs[8])
    assert out.dtype == dtype and last.dtype == torch.float32
    check("out", out, rout)
    check("last state", last, rlast)
    got = _grads([out, last], [g, glast], leaves)
    want = _grads([rout, rlast], [g.double(), glast.double()], refs)
    for name, a, r in zip((*ORDER, "initial_state"), got, want):
        check(f"gradient of {name}", a, r)
    with torch.no_grad():  # without gradients: the same values, no states kept
        assert torch.equal(sg.selective_scan(*leaves[:8], initial_state=leaves[8]), out)


@pytest.mark.parametrize("b,t,c,n", [(1, 700, 96, 16), (2, 1029, 40, 16), (1, 520, 200, 8), (24, 300, 130, 16)])
def test_scan_long_sequences(cuda, b, t, c, n):
    """Lengths and batches at which the work is split over time, and where it is not."""
    ins, h0, g = scan_inputs(b, t, c, n, torch.float32, cuda, seed=3)
    glast = torch.randn(h0.shape, generator=torch.Generator().manual_seed(1)).to(cuda)
    leaves = [ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True)
    refs = [wide(v) for v in leaves]
    rout, rlast = scan_ref(*refs[:8], h0=refs[8])
    check("out", out, rout)
    check("last state", last, rlast)
    got = _grads([out, last], [g, glast], leaves)
    want = _grads([rout, rlast], [g.double(), glast.double()], refs)
    for name, a, r in zip((*ORDER, "initial_state"), got, want):
        check(f"gradient of {name}", a, r)
    with torch.no_grad():
        out2, last2 = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True)
    check("out without gradients", out2, rout)
    check("last state without gradients", last2, rlast)


@pytest.mark.parametrize("missing", ["D", "z", "dt_bias", "all"])
def test_scan_without_the_optional_inputs(cuda, missing):
    ins, _, g = scan_inputs(2, 21, 37, 16, torch.float32, cuda, seed=5)
    for k in ("D", "z", "dt_bias"):
        if missing in (k, "all"):
            ins[k] = None
    ins["dt"] = ins["dt"].abs() * 0.1  # softplus off: the step as it is
    for softplus in (True, False):
        leaves = [None if ins[k] is None else ins[k].detach().requires_grad_() for k in ORDER]
        if not softplus and leaves[7] is not None:
            leaves[7] = leaves[7].detach().abs().mul(0.1).requires_grad_()
        refs = [wide(v) for v in leaves]
        out = sg.selective_scan(*leaves, dt_softplus=softplus)
        rout, _ = scan_ref(*refs, softplus=softplus)
        check("out", out, rout)
        has = [i for i, v in enumerate(leaves) if v is not None]
        got = _grads([out], [g], [leaves[i] for i in has])
        want = _grads([rout], [g.double()], [refs[i] for i in has])
        for i, a, r in zip(has, got, want):
            check(f"gradient of {ORDER[i]}", a, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,c", [(37, 48), (530, 33)])
def test_scan_right_padded_batch_reads_no_padding(cuda, dtype, t, c):
    ins, h0, g = scan_inputs(5, t, c, 16, dtype, cuda, seed=7)
    lengths = torch.tensor([0, 1, t, t - 9, 16], device=cuda)
    past = torch.arange(t, device=cuda)[None] >= lengths[:, None]
    ref_in = {k: v.clone() for k, v in ins.items()}
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=cuda).to(dtype)
    for i, k in enumerate(("x", "dt", "B", "C", "z")):
        ins[k][past] = bad[i % 3]
    g = torch.where(past[..., None], torch.full_like(g, float("nan")), g)
    leaves = [ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    refs = [wide(ref_in[k]) for k in ORDER] + [wide(h0)]
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], lengths=lengths, return_state=True)
    rout, rlast = scan_ref(*refs[:8], h0=refs[8], lengths=lengths)
    check("out", out, rout)
    check("last state", last, rlast)
    assert (out[past] == 0).all() and torch.equal(last[0], h0[0])
    glast = torch.ones_like(last)
    got = _grads([out, last], [g, glast], leaves)
    gref = torch.where(past[..., None], torch.zeros_like(g), g).double()
    want = _grads([rout, rlast], [gref, glast.double()], refs)
    for name, a, r in zip((*ORDER, "initial_state"), got, want):
        check(f"gradient of {name}", a, r)


def test_scan_reads_slices_of_wider_projections_in_place(cuda):
    """x, z as halves of one tensor; dt, B, C as parts of another, at odd offsets and
    pitches; a transposed input; an expanded gradient."""
    b, t, c, n = 2, 45, 52, 16
    gen = torch.Generator().manual_seed(9)
    for dtype in (torch.float32, torch.bfloat16):
        xz = torch.randn(b, t, 2 * c + 3, generator=gen).to(cuda, dtype)
        low = (torch.randn(b, t, c + 2 * n + 1, generator=gen) * 0.5).to(cuda, dtype)
        A, D, bias = -torch.rand(c, n, generator=gen).to(cuda) * 4, torch.ones(c, device=cuda), torch.zeros(c, device=cuda)
        views = dict(x=xz[..., :c], z=xz[..., c + 3 :], dt=low[..., 1 : c + 1], B=low[..., c + 1 : c + 1 + n],
                     C=low[..., c + 1 + n :])
        args = [views["x"], views["dt"], A, views["B"], views["C"], D, views["z"], bias]
        want = sg.selective_scan(*[a.contiguous() for a in args])
        assert torch.equal(sg.selective_scan(*args), want)
        flipped = [a.transpose(0, 1).contiguous().transpose(0, 1) if a.ndim == 3 else a for a in args]
        assert torch.equal(sg.selective_scan(*flipped), want)
        channels_first = [a.transpose(1, 2).contiguous().transpose(1, 2) if a.ndim == 3 else a for a in args]
        assert torch.equal(sg.selective_scan(*channels_first), want)
        leaf = [a.detach().requires_grad_() for a in args]
        got = _grads([sg.selective_scan(*leaf).float().sum()], None, leaf)
        plain = [a.detach().contiguous().requires_grad_() for a in args]
        ref = _grads([sg.selective_scan(*plain).float().sum()], None, plain)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("where", ["x", "dt", "z", "gradient"])
@pytest.mark.parametrize("n", [3, 8, 16, 24, 64])
def test_scan_infinities_stay_in_their_channel(cuda, n, where, value):
    """A value that is not finite reaches its own sequence's channel and the sums over
    channels, and no other channel's outputs and gradients."""
    b, t, c, hit = 2, 45, 70, 21
    ins, _, g = scan_inputs(b, t, c, n, torch.float32, cuda, seed=9)
    refs = {k: wide(v) for k, v in ins.items()}
    rout, _ = scan_ref(*[refs[k] for k in ORDER])
    want = dict(zip(ORDER, _grads(rout, g.double(), [refs[k] for k in ORDER])))
    spoilt = {k: v.clone() for k, v in ins.items()}
    g = g.clone()
    (g if where == "gradient" else spoilt[where])[1, 30, hit] = value
    leaves = [spoilt[k].requires_grad_() for k in ORDER]
    out = sg.selective_scan(*leaves)
    got = dict(zip(ORDER, _grads(out, g, leaves)))
    others = torch.arange(c, device=cuda) != hit
    check("out", out[..., others], rout[..., others])
    check("out of the other sequence", out[0], rout[0])
    for k in ("x", "dt", "z"):
        check(f"gradient of {k}", got[k][..., others], want[k][..., others])
        check(f"gradient of {k} in the other sequence", got[k][0], want[k][0])
    for k in ("A", "D", "dt_bias"):
        check(f"gradient of {k}", got[k][others], want[k][others])
    for k in ("B", "C"):
        check(f"gradient of {k} in the other sequence", got[k][0], want[k][0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_split_sequence_and_empty_sequence(cuda, dtype):
    ins, h0, _ = scan_inputs(2, 90, 41, 16, dtype, cuda, seed=11)
    seq = ("x", "dt", "B", "C", "z")
    whole, last = sg.selective_scan(*[ins[k] for k in ORDER], initial_state=h0, return_state=True)
    state, parts = h0, []
    for lo, hi in ((0, 0), (0, 1), (1, 50), (50, 90)):
        cut = {k: (v[:, lo:hi] if k in seq else v) for k, v in ins.items()}
        y, state = sg.selective_scan(*[cut[k] for k in ORDER], initial_state=state, return_state=True)
        parts.append(y)
        if hi == 0:
            assert torch.equal(state, h0)
    check("joined out", torch.cat(parts, 1), whole.double())
    check("joined state", state, last.double())
    _, s = sg.selective_scan(*[(v[:, :0] if k in seq else v) for k, v in ((k, ins[k]) for k in ORDER)],
                             return_state=True)
    assert (s == 0).all()


def test_scan_empty_sequence_has_gradients(cuda):
    ins, h0, _ = scan_inputs(2, 0, 20, 16, torch.float32, cuda)
    leaves = [ins[k].requires_grad_() for k in ORDER] + [h0.requires_grad_()]
    out, last = sg.selective_scan(*leaves[:8], initial_state=leaves[8], return_state=True)
    got = _grads([out.sum() + (last * 3).sum()], None, leaves)
    assert (got[8] == 3).all()
    for name, v in zip(ORDER, got[:8]):
        assert v is not None and (v == 0).all(), name


def test_scan_gradient_against_differences(cuda):
    """Directional derivatives of the kernel's own forward: with a step of 1e-2 the
    central difference is off by its square times the third derivative (about 1e-4
    of the value) and by the float32 noise of the outputs over the step (1e-4)."""
    ins, h0, g = scan_inputs(2, 40, 35, 16, torch.float32, cuda, seed=13)
    args = {**ins, "initial_state": h0}
    names = (*ORDER, "initial_state")

    def loss(a):
        out = sg.selective_scan(*[a[k] for k in ORDER], initial_state=a["initial_state"])
        return (out.double() * g.double()).sum()

    leaves = {k: v.detach().requires_grad_() for k, v in args.items()}
    out = sg.selective_scan(*[leaves[k] for k in ORDER], initial_state=leaves["initial_state"])
    grads = dict(zip(names, _grads([out], [g], [leaves[k] for k in names])))
    for k in names:
        v = grads[k].sign()  # the loss grows along it, and no element moves further than the step
        eps = 1e-2 * float(args[k].abs().mean().clamp(min=0.1))
        with torch.no_grad():
            up = loss({**args, k: args[k] + eps * v})
            down = loss({**args, k: args[k] - eps * v})
        numeric = float(up - down) / (2 * eps)
        exact = float((grads[k].double() * v.double()).sum())
        assert abs(numeric - exact) <= 5e-3 * abs(exact), (k, numeric, exact)


def test_scan_strong_decay_and_large_steps(cuda):
    """A decay that underflows to zero, steps past softplus's linear end, and gates
    at their limits give finite values that match."""
    ins, h0, g = scan_inputs(2, 50, 38, 16, torch.float32, cuda, seed=17)
    ins["A"] = ins["A"] * 50
    ins["dt"][:, ::5] += 40
    ins["dt"][:, 1::7] -= 60
    ins["z"][:, ::3] *= 30
    leaves = [ins[k].requires_grad_() for k in ORDER]
    refs = [wide(v) for v in leaves]
    out, rout = sg.selective_scan(*leaves), scan_ref(*refs)[0]
    check("out", out, rout)
    for name, a, r in zip(ORDER, _grads([out], [g], leaves), _grads([rout], [g.double()], refs)):
        check(f"gradient of {name}", a, r)


def test_scan_is_deterministic(cuda):
    ins, h0, g = scan_inputs(3, 333, 200, 16, torch.bfloat16, cuda, seed=19)
    leaves = [ins[k].requires_grad_() for k in ORDER]
    runs = []
    for _ in range(2):
        out = sg.selective_scan(*leaves)
        runs.append([out, *_grads([out], [g], leaves)])
    assert all(torch.equal(p, q) for p, q in zip(*runs))


def test_scan_on_another_stream_and_in_a_graph(cuda):
    ins, h0, _ = scan_inputs(2, 64, 64, 16, torch.bfloat16, cuda, seed=23)
    args = [ins[k] for k in ORDER]
    want = sg.selective_scan(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sg.selective_scan(*args)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = sg.selective_scan(*args)
    args[0].mul_(2)
    graph.replay()
    assert torch.equal(held, sg.selective_scan(*args))


def test_scan_and_conv_compile_fullgraph(cuda):
    ins, _, g = scan_inputs(2, 30, 24, 8, torch.float32, cuda, seed=29)
    w, bias = torch.randn(24, 4, device=cuda), torch.randn(24, device=cuda)

    def f(x, dt, A, B, C, D, z, dt_bias, w, bias):
        u = sg.causal_conv(x, w, bias)
        out, last = sg.selective_scan(u, dt, A, B, C, D, z, dt_bias, return_state=True)
        return sg.layer_norm(out, D, dt_bias), last

    args = [ins[k].requires_grad_() for k in ORDER] + [w.requires_grad_(), bias.requires_grad_()]
    eager = f(*args)
    compiled = torch.compile(f, fullgraph=True)(*args)
    assert torch.equal(eager[0], compiled[0]) and torch.equal(eager[1], compiled[1])
    for p, q in zip(_grads([eager[0]], [g], args), _grads([compiled[0]], [g], args)):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,c,n", [(1, 64, 16), (3, 37, 16), (2, 130, 8), (5, 20, 5), (2, 24, 64), (1, 1, 1), (70, 48, 16)])
def test_scan_step_is_one_token_of_the_scan(cuda, dtype, b, c, n):
    ins, h0, _ = scan_inputs(b, 3, c, n, dtype, cuda, seed=31)
    seq = ("x", "dt", "B", "C", "z")
    out, last = scan_ref(*[ins[k].double() for k in ORDER], h0=h0.double())
    state = h0.clone()
    for t in range(3):
        one = {k: (ins[k][:, t] if k in seq else ins[k]) for k in ORDER}
        y = sg.selective_scan_step_(one["x"], one["dt"], one["A"], one["B"], one["C"], state, one["D"], one["z"],
                                    one["dt_bias"])
        check(f"token {t}", y, out[:, t])
    check("state", state, last)
    plain = h0.clone()
    y = sg.selective_scan_step_(ins["x"][:, 0], ins["dt"][:, 0].abs(), ins["A"], ins["B"][:, 0], ins["C"][:, 0], plain,
                                dt_softplus=False)
    ref, rl = scan_ref(*[ins[k][:, :1].double() if k in seq else ins[k].double() for k in ("x",)],
                       ins["dt"][:, :1].double().abs(), ins["A"].double(), ins["B"][:, :1].double(),
                       ins["C"][:, :1].double(), h0=h0.double(), softplus=False)
    check("plain token", y, ref[:, 0])
    check("plain state", plain, rl)


# -------------------------------------------------------------- convolution


def _conv_inputs(b, t, c, w, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed + b + 3 * t + 5 * c + 7 * w)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return (n(b, t, c).to(device, dtype), (n(c, w) / w**0.5).to(device), (n(c) * 0.2).to(device),
            n(b, w - 1, c).to(device, dtype), n(b, t, c).to(device, dtype))  # fmt: skip


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("w", [1, 2, 3, 4])
@pytest.mark.parametrize("b,t,c", [(1, 1, 1), (2, 3, 64), (3, 65, 37), (1, 200, 136), (2, 32, 258), (1, 33, 1028)])
def test_conv_outputs_and_gradients(cuda, b, t, c, w, dtype):
    for silu in (True, False):
        x, weight, bias, window, g = _conv_inputs(b, t, c, w, dtype, cuda)
        leaves = [v.requires_grad_() for v in (x, weight, bias, window)]
        refs = [wide(v) for v in leaves]
        y, state = sg.causal_conv(x, weight, bias, silu=silu, initial_state=window, return_state=True)
        ry, rstate = conv_ref(*refs, silu=silu)
        check("y", y, ry)
        assert torch.equal(state.double(), rstate)
        gs = torch.ones_like(state)
        got = _grads([y, state], [g, gs], leaves)
        want = _grads([ry, rstate], [g.double(), gs.double()], refs)
        for name, a, r in zip(("x", "weight", "bias", "window"), got, want):
            if r is None or r.numel() == 0:
                continue
            if name in ("x", "window") and dtype != torch.float32:
                # the state's gradient of ones is added in the tensor's type: one more rounding
                torch.testing.assert_close(a.double(), r, rtol=2**-6, atol=2e-2)
            else:
                check(f"gradient of {name}", a, r)
        got = _grads([sg.causal_conv(x, weight, None, silu=silu)], [g], leaves[:2])
        want = _grads([conv_ref(refs[0], refs[1], None, silu=silu)[0]], [g.double()], refs[:2])
        for name, a, r in zip(("x", "weight"), got, want):
            check(f"gradient of {name} alone", a, r)
        with torch.no_grad():
            y2, s2 = sg.causal_conv(x, weight, bias, silu=silu, initial_state=window, return_state=True)
        assert torch.equal(y2, y) and torch.equal(s2, state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [48, 33])
def test_conv_right_padded_batch_reads_no_padding(cuda, dtype, c):
    t = 70
    x, weight, bias, window, g = _conv_inputs(5, t, c, 4, dtype, cuda, seed=3)
    lengths = torch.tensor([0, 2, t, 33, 64], device=cuda, dtype=torch.int32)
    past = (torch.arange(t, device=cuda)[None] >= lengths[:, None])[..., None]
    refs = [wide(v) for v in (x, weight, bias, window)]
    x = torch.where(past, torch.full_like(x, float("nan")), x)
    leaves = [v.requires_grad_() for v in (x, weight, bias, window)]
    y = sg.causal_conv(x, weight, bias, initial_state=window, lengths=lengths)
    ry, rstate = conv_ref(*refs, lengths=lengths)
    check("y", y, ry)
    gnan = torch.where(past, torch.full_like(g, float("nan")), g)
    gzero = torch.where(past, torch.zeros_like(g), g).double()
    for name, a, r in zip(("x", "weight", "bias", "window"), _grads([y], [gnan], leaves), _grads([ry], [gzero], refs)):
        check(f"gradient of {name}", a, r)
    with torch.no_grad():
        y2, state = sg.causal_conv(x, weight, bias, initial_state=window, lengths=lengths, return_state=True)
    assert torch.equal(y2, y) and torch.equal(state.double(), rstate)
    _, state = sg.causal_conv(x, weight, bias, initial_state=window, lengths=lengths, return_state=True)
    assert torch.equal(state.double(), rstate)


def test_conv_infinities_stay_within_their_reach(cuda):
    """A tap outside the width must not see a row: rows W or more before stay out."""
    x, weight, bias, _, _ = _conv_inputs(1, 40, 24, 2, torch.float32, cuda, seed=5)
    x[0, 10] = float("inf")
    x[0, 20] = float("nan")
    y = sg.causal_conv(x, weight, bias, silu=False)
    touched = torch.zeros(40, dtype=torch.bool, device=cuda)
    touched[[10, 11, 20, 21]] = True
    assert torch.isfinite(y[0, ~touched]).all() and not torch.isfinite(y[0, touched]).any()


def test_conv_strides_split_and_empty(cuda):
    for dtype in (torch.float32, torch.bfloat16):
        x, weight, bias, window, _ = _conv_inputs(2, 77, 44, 4, dtype, cuda, seed=7)
        want, last = sg.causal_conv(x, weight, bias, initial_state=window, return_state=True)
        holder = torch.full((2, 77, 51), float("nan"), dtype=dtype, device=cuda)
        holder[..., 5:49] = x
        assert torch.equal(sg.causal_conv(holder[..., 5:49], weight, bias, initial_state=window), want)
        assert torch.equal(sg.causal_conv(x.transpose(0, 1).contiguous().transpose(0, 1), weight, bias,
                                          initial_state=window), want)
        state, parts = window, []
        for lo, hi in ((0, 0), (0, 1), (1, 3), (3, 40), (40, 77)):
            y, state = sg.causal_conv(x[:, lo:hi], weight, bias, initial_state=state, return_state=True)
            parts.append(y)
        assert torch.equal(torch.cat(parts, 1), want) and torch.equal(state, last)
    xe = torch.zeros(2, 0, 44, device=cuda, requires_grad=True)
    w = weight.detach().requires_grad_()
    gx, gw = _grads([sg.causal_conv(xe, w, bias).sum()], None, [xe, w])
    assert gx.shape == xe.shape and (gw == 0).all()


def test_conv_gradient_against_differences(cuda):
    x, weight, bias, window, g = _conv_inputs(2, 30, 36, 4, torch.float32, cuda, seed=9)
    args = [x, weight, bias, window]

    def loss(a):
        return (sg.causal_conv(a[0], a[1], a[2], initial_state=a[3]).double() * g.double()).sum()

    leaves = [v.detach().requires_grad_() for v in args]
    grads = _grads([sg.causal_conv(*leaves[:3], initial_state=leaves[3])], [g], leaves)
    for i, name in enumerate(("x", "weight", "bias", "window")):
        v = grads[i] / grads[i].abs().mean()
        with torch.no_grad():
            up = loss([a + 5e-3 * v if j == i else a for j, a in enumerate(args)])
            down = loss([a - 5e-3 * v if j == i else a for j, a in enumerate(args)])
        numeric, exact = float(up - down) / 1e-2, float((grads[i].double() * v.double()).sum())
        assert abs(numeric - exact) <= 5e-3 * abs(exact), (name, numeric, exact)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("w", [1, 2, 3, 4])
@pytest.mark.parametrize("b,c", [(1, 64), (3, 37), (70, 130), (1, 1)])
def test_conv_step_is_one_token_of_the_convolution(cuda, dtype, w, b, c):
    x, weight, bias, window, _ = _conv_inputs(b, 5, c, w, dtype, cuda, seed=11)
    ry, rstate = conv_ref(x.double(), weight.double(), bias.double(), window.double())
    state = window.clone()
    for t in range(5):
        check(f"token {t}", sg.causal_conv_step_(x[:, t], state, weight, bias), ry[:, t])
    assert torch.equal(state.double(), rstate)
    state = window.clone()
    y = sg.causal_conv_step_(x[:, 0], state, weight, silu=False)
    check("plain token", y, conv_ref(x[:, :1].double(), weight.double(), None, window.double(), silu=False)[0][:, 0])


# ---------------------------------------------------------------- refusals


def test_refusals(cuda):
    ins, h0, _ = scan_inputs(2, 8, 16, 4, torch.float32, cuda)
    base = [ins[k] for k in ORDER]

    def scan(**change):
        a = {**ins, **{k: v for k, v in change.items() if k in ORDER}}
        return sg.selective_scan(*[a[k] for k in ORDER], **{k: v for k, v in change.items() if k not in ORDER})

    for bad in (dict(x=ins["x"][0]), dict(x=ins["x"].double()), dict(dt=ins["dt"][:, :4]), dict(B=ins["B"].half()),
                dict(C=ins["C"][..., :3]), dict(A=ins["A"][:8]), dict(A=torch.zeros(16, 65, device=cuda)),
                dict(A=torch.zeros(16, 0, device=cuda)), dict(D=ins["D"][:3]), dict(dt_bias=ins["D"][:3]),
                dict(z=ins["z"][:1]), dict(initial_state=h0[:1]), dict(initial_state=h0.half()),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device=cuda)), dict(lengths=torch.zeros(2, device=cuda)),
                dict(D=ins["D"].cpu())):  # fmt: skip
        with pytest.raises(ValueError):
            scan(**bad)
    with pytest.raises(NotImplementedError):
        sg.selective_scan(*[v.cpu() for v in base])
    step = [ins["x"][:, 0], ins["dt"][:, 0], ins["A"], ins["B"][:, 0], ins["C"][:, 0]]
    for state in (h0.half(), h0[:1], h0.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError):
            sg.selective_scan_step_(*step, state)
    with pytest.raises(ValueError):
        sg.selective_scan_step_(ins["x"], *step[1:], h0)
    with pytest.raises(ValueError):
        sg.selective_scan_step_(*step[:3], ins["B"][:, 0].half(), step[4], h0)
    with pytest.raises(NotImplementedError):
        sg.selective_scan_step_(step[0].clone().requires_grad_(), *step[1:], h0.clone())
    x, w = torch.zeros(2, 8, 16, device=cuda), torch.zeros(16, 4, device=cuda)
    for args, kw in (((x[0], w), {}), ((x, w[:3]), {}), ((x, torch.zeros(16, 5, device=cuda)), {}), ((x, w, w[:, 0][:3]), {}),
                     ((x, w), dict(initial_state=torch.zeros(2, 4, 16, device=cuda))),
                     ((x, w), dict(initial_state=torch.zeros(2, 3, 16, device=cuda).half())), ((x.long(), w), {})):  # fmt: skip
        with pytest.raises(ValueError):
            sg.causal_conv(*args, **kw)
    with pytest.raises(ValueError):
        sg.causal_conv_step_(x[:, 0], torch.zeros(2, 16, 3, device=cuda).transpose(1, 2), w)
    with pytest.raises(ValueError):
        sg.causal_conv_step_(x, torch.zeros(2, 3, 16, device=cuda), w)
    lib, p = _capi.lib(), x.data_ptr()
    assert lib.causal_conv_forward(1, p, p, None, None, None, p, None, 2, 8, 16, 5, 128, 16, 1, None) == 1
    assert lib.selective_scan_step(0, p, p, p, p, p, p, None, None, None, p, 1, 4, 65, 4, 4, 4, 4, 0, 1, None) == 1


def test_kernels_are_counted(cuda):
    before = _capi.launch_counts()
    ins, h0, g = scan_inputs(1, 20, 16, 16, torch.float32, cuda)
    leaves = [ins[k].requires_grad_() for k in ORDER]
    _grads([sg.selective_scan(*leaves)], [g], leaves)
    w = torch.zeros(16, 4, device=cuda, requires_grad=True)
    _grads([sg.causal_conv(ins["x"], w).sum()], None, [w])
    with torch.no_grad():
        sg.causal_conv_step_(ins["x"][:, 0], torch.zeros(1, 3, 16, device=cuda), w)
        sg.selective_scan_step_(*[ins[k][:, 0] if k != "A" else ins[k] for k in ORDER[:5]], h0)
    after = _capi.launch_counts()
    for k in ("scan_fwd_kernel", "scan_bwd_kernel", "scan_reduce_kernel", "column_sum_kernel", "causal_conv_fwd_kernel",
              "causal_conv_bwd_kernel", "causal_conv_step_kernel", "scan_step_kernel"):  # fmt: skip
        assert after[k] > before[k], k
