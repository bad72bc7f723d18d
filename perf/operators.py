"""Cases of the selective-mixer operators: the short causal convolution, the selective scan, their single-token
steps, layer norm, and the matrix-vector product with 4-bit weights.

``run`` computes one pass through an operator, in plain torch operations (``own`` false) or through the
package's public entry points (``own`` true). ``exact`` is the operator's definition in 64 bits."""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _package():
    where = os.path.join(_ROOT, "spikegpt-myelin_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    import spikegpt_b200

    return spikegpt_b200


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # training the short convolution: 8 sequences of 1024 tokens, inner width 2 x 512 (the 41M configuration's width)
        {"name": "conv train 8x1024x1024", "kind": "conv_train", "b": 8, "t": 1024, "c": 1024, "w": 4, "type": "bf16"},
        # prompts of several lengths in one right-padded batch, continued from a cached window, in float32
        {"name": "conv prompt 5x1003x1536", "kind": "conv_prompt", "b": 5, "t": 1003, "c": 1536, "w": 4, "type": "f32", "ragged": True},
        # training the scan with few sequences: one GPU's share of a small global batch
        {"name": "scan train 2x1024x1024", "kind": "scan_train", "b": 2, "t": 1024, "c": 1024, "n": 16, "type": "bf16"},
        # training the scan at a full batch, inner width 2 x 768 (the 216M configuration's width)
        {"name": "scan train 16x1024x1536", "kind": "scan_train", "b": 16, "t": 1024, "c": 1536, "n": 16, "type": "bf16"},
        # training in float32 at odd sizes: a ragged last tile in time and in channels, 12 states
        {"name": "scan train 3x333x523", "kind": "scan_train", "b": 3, "t": 333, "c": 523, "n": 12, "type": "f32"},
        # one long prompt of odd length, whose final state starts the generation
        {"name": "scan prompt 1x8191x1536", "kind": "scan_prompt", "b": 1, "t": 8191, "c": 1536, "n": 16, "type": "bf16", "ragged": False},
        # one token for one sequence, the convolution's step and the scan's: latency counts
        {"name": "step 1x1024", "kind": "step", "b": 1, "c": 1024, "n": 16, "w": 4, "type": "bf16"},
        # one token for each of 256 sequences: the state's traffic counts
        {"name": "step 256x1536", "kind": "step", "b": 256, "c": 1536, "n": 16, "w": 4, "type": "bf16"},
        # the norm of a float32 residual stream, 8 x 1024 tokens of width 512
        {"name": "norm train 8192x512", "kind": "norm_train", "rows": 8192, "c": 512, "type": "f32"},
        # the norm of a wide bf16 model's training batch
        {"name": "norm train 16384x4096", "kind": "norm_train", "rows": 16384, "c": 4096, "type": "bf16"},
        # the output head of the 216M configuration for one token
        {"name": "matvec 1x768x50257", "kind": "matvec", "m": 1, "k": 768, "n": 50257, "g": 64, "type": "bf16"},
        # a wide model's up-projection for a handful of sequences
        {"name": "matvec 6x8192x16384", "kind": "matvec", "m": 6, "k": 8192, "n": 16384, "g": 128, "type": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["conv_train", "conv_prompt", "scan_train", "scan_train", "scan_prompt", "step", "norm_train", "matvec"])
    kinds = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "matvec":
        k = _spread(rng, 100, 8192)
        k = k if rng.random() < 0.4 else -(-k // 64) * 64
        n = min(_spread(rng, 100, 50257), 16384 * 8192 // k)
        return {"kind": kind, "m": rng.randint(1, 6), "k": k, "n": n, "g": rng.choice([32, 64, 128]), "type": kinds}
    if kind == "norm_train":
        c = _spread(rng, 33, 8192)
        return {"kind": kind, "rows": min(_spread(rng, 1, 16384), 16384 * 4096 // (2 if kinds == "f32" else 1) // c), "c": c, "type": kinds}
    if kind == "step":
        return {"kind": kind, "b": _spread(rng, 1, 256), "c": _spread(rng, 64, 1536), "n": rng.choice([8, 16, 16]), "w": rng.randint(2, 4), "type": kinds}
    c = _spread(rng, 64, 1536)
    if kind == "scan_prompt":
        t = _spread(rng, 1, 8191)
        return {"kind": kind, "b": max(1, min(_spread(rng, 1, 16), 8191 // t)), "t": t, "c": c, "n": rng.choice([8, 16, 16]), "type": kinds, "ragged": rng.random() < 0.5}
    if kind == "scan_train":
        return {"kind": kind, "b": rng.randint(1, 16), "t": _spread(rng, 1, 1024), "c": c, "n": rng.choice([8, 13, 16, 16]), "type": kinds}
    t = _spread(rng, 1, 1024)
    case = {"kind": kind, "b": max(1, min(rng.randint(1, 8), 8 * 1024 * 512 // (t * c))), "t": t, "c": c, "w": rng.randint(2, 4), "type": kinds}
    if kind == "conv_prompt":
        case["ragged"] = rng.random() < 0.5
    return case


def work(case):
    kind, e = case["kind"], _SIZES[case["type"]]
    if kind == "matvec":
        groups = -(-case["k"] // case["g"])
        size = case["n"] * (case["k"] / 2 + groups * 3) + case["m"] * (case["k"] + case["n"]) * e
        return {"bytes": size, "flops": 2 * case["m"] * case["n"] * case["k"]}
    if kind == "norm_train":
        cells = case["rows"] * case["c"]
        return {"bytes": 5 * e * cells + 16 * case["c"], "flops": 20 * cells}
    if kind == "step":
        cells = case["b"] * case["c"]
        size = cells * (8 * case["n"] + 2 * (case["w"] - 1) * e + 6 * e) + case["c"] * 4 * (case["n"] + case["w"] + 3) + 2 * case["b"] * case["n"] * e
        return {"bytes": size, "flops": cells * (7 * case["n"] + 2 * case["w"] + 20)}
    cells = case["b"] * case["t"] * case["c"]
    if kind == "conv_train":
        return {"bytes": 5 * e * cells + 8 * case["c"] * (case["w"] + 1), "flops": cells * (8 * case["w"] + 20)}
    if kind == "conv_prompt":
        return {"bytes": 2 * e * cells + 4 * case["c"] * (case["w"] + 1), "flops": cells * (2 * case["w"] + 8)}
    rows = case["b"] * case["t"] * case["n"]
    states = case["b"] * case["c"] * case["n"]
    if kind == "scan_prompt":
        return {"bytes": 4 * e * cells + 2 * e * rows + 8 * states + 4 * case["c"] * (case["n"] + 2), "flops": cells * (7 * case["n"] + 20)}
    return {"bytes": 11 * e * cells + 6 * e * rows + 8 * case["c"] * (case["n"] + 2), "flops": cells * (24 * case["n"] + 50)}


# ------------------------------------------------------------------ the inputs


class _Maker:
    def __init__(self, seed):
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.rng = torch.Generator(device=self.device).manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, shift=0.0, kind=torch.float32):
        v = torch.randn(shape, generator=self.rng, device=self.device)
        return (v * scale + shift).to(kind)

    def uniform(self, *shape, low=0.0, high=1.0):
        return torch.rand(shape, generator=self.rng, device=self.device) * (high - low) + low

    def whole(self, low, high, shape, kind):
        return torch.randint(low, high, shape, generator=self.rng, device=self.device, dtype=kind)


def _scan_parameters(make, c, n):
    """A near -1 .. -n, and a bias whose softplus lies in 0.001 .. 0.1: the usual start of such models."""
    a = -torch.arange(1, n + 1, device=make.device, dtype=torch.float32) * torch.exp(0.1 * make.normal(c, n))
    step = torch.exp(make.uniform(c, low=math.log(1e-3), high=math.log(1e-1)))
    return {"A": a, "D": make.normal(c, scale=0.1, shift=1.0), "dt_bias": step + torch.log(-torch.expm1(-step))}


def _inputs(case, seed):
    kind, form, make = case["kind"], _TYPES[case["type"]], _Maker(seed)
    if kind == "matvec":
        m, k, n, g = case["m"], case["k"], case["n"], case["g"]
        padded = -(-k // 32) * 32
        return {
            "x": make.normal(m, k, kind=form),
            "packed": make.whole(0, 256, (n, padded // 2), torch.uint8),
            "scales": (make.uniform(n, -(-k // g), low=0.5, high=1.5) / (4.6 * math.sqrt(k))).to(torch.bfloat16),
            "zeros": make.whole(6, 11, (n, -(-k // g)), torch.uint8),
        }
    c = case["c"]
    if kind == "norm_train":
        rows = case["rows"]
        return {
            "x": (make.normal(rows, c, scale=2.0) + make.normal(rows, 1)).to(form),
            "weight": make.normal(c, scale=0.2, shift=1.0),
            "bias": make.normal(c, scale=0.2),
            "grad": make.normal(rows, c, kind=form),
        }
    b = case["b"]
    taps = {}
    if "w" in case:
        taps = {"weight": make.normal(c, case["w"], scale=case["w"] ** -0.5), "bias": make.normal(c, scale=0.1)}
    if kind == "step":
        n = case["n"]
        return {
            "x": make.normal(b, c, kind=form), "u": make.normal(b, c, kind=form),
            "dt": make.normal(b, c, scale=0.5, kind=form), "z": make.normal(b, c, kind=form),
            "B": make.normal(b, n, kind=form), "C": make.normal(b, n, kind=form),
            "window": make.normal(b, case["w"] - 1, c, kind=form), "state": make.normal(b, c, n, scale=0.3),
            **taps, **_scan_parameters(make, c, n),
        }
    t = case["t"]
    got = {"x": make.normal(b, t, c, kind=form), **taps}
    if case.get("ragged"):
        got["lengths"] = make.whole(0, t + 1, (b,), torch.int32)
    if kind == "conv_train":
        return {**got, "grad": make.normal(b, t, c, kind=form)}
    if kind == "conv_prompt":
        return {**got, "window": make.normal(b, case["w"] - 1, c, kind=form)}
    n = case["n"]
    got |= {"dt": make.normal(b, t, c, scale=0.5, kind=form), "z": make.normal(b, t, c, kind=form)}
    got |= {"B": make.normal(b, t, n, kind=form), "C": make.normal(b, t, n, kind=form), **_scan_parameters(make, c, n)}
    if kind == "scan_prompt":
        return {**got, "state": make.normal(b, c, n, scale=0.3)}
    return {**got, "grad": make.normal(b, t, c, kind=form)}


_LEARNED = {
    "conv_train": ("x", "weight", "bias"),
    "norm_train": ("x", "weight", "bias"),
    "scan_train": ("x", "dt", "A", "B", "C", "D", "z", "dt_bias"),
}


def prepare(case, seed):
    state = _inputs(case, seed)
    for name in _LEARNED.get(case["kind"], ()):
        state[name].requires_grad_()
    return {"case": dict(case), **state}


# ------------------------------------------------------------------ one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    with torch.no_grad():
        return _PLAIN[kind](state)


def _own_conv_train(s):
    y = _package().causal_conv(s["x"], s["weight"], s["bias"])
    return [y.detach(), *torch.autograd.grad(y, [s[k] for k in _LEARNED["conv_train"]], s["grad"])]


def _own_conv_prompt(s):
    return list(_package().causal_conv(s["x"], s["weight"], s["bias"], initial_state=s["window"], lengths=s.get("lengths"), return_state=True))


def _own_scan_train(s):
    y = _package().selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"])
    return [y.detach(), *torch.autograd.grad(y, [s[k] for k in _LEARNED["scan_train"]], s["grad"])]


def _own_scan_prompt(s):
    return list(
        _package().selective_scan(
            s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"],
            initial_state=s["state"], lengths=s.get("lengths"), return_state=True,
        )
    )  # fmt: skip


def _own_step(s):
    p = _package()
    v = p.causal_conv_step_(s["x"], s["window"], s["weight"], s["bias"])
    y = p.selective_scan_step_(s["u"], s["dt"], s["A"], s["B"], s["C"], s["state"], s["D"], s["z"], s["dt_bias"])
    return [v, y, s["window"], s["state"]]


def _own_norm_train(s):
    y = _package().layer_norm(s["x"], s["weight"], s["bias"], 1e-5)
    return [y.detach(), *torch.autograd.grad(y, [s[k] for k in _LEARNED["norm_train"]], s["grad"])]


def _own_matvec(s):
    return _package().q4_linear(s["x"], s["packed"], s["scales"], s["zeros"], group_size=s["case"]["g"])


_OWN = {
    "conv_train": _own_conv_train, "conv_prompt": _own_conv_prompt, "scan_train": _own_scan_train, "scan_prompt": _own_scan_prompt,
    "step": _own_step, "norm_train": _own_norm_train, "matvec": _own_matvec,
}  # fmt: skip


# ------------------------------------------------------------------ the plain forms


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _windows(x, front, w):
    """[B, T, C, W]: each row with the W - 1 rows before it."""
    return torch.cat([front, x], 1).unfold(1, w, 1)


def _valid(s):
    """[B, T, 1]: which rows lie inside their sequence."""
    t = s["x"].shape[1]
    if "lengths" not in s:
        return torch.ones((1, t, 1), dtype=torch.bool, device=s["x"].device)
    return (torch.arange(t, device=s["x"].device)[None, :] < s["lengths"][:, None])[..., None]


def _plain_conv_train(s):
    x, grad, weight = s["x"].float(), s["grad"].float(), s["weight"]
    b, _, c = x.shape
    w = weight.shape[1]
    edge = x.new_zeros(b, w - 1, c)
    seen = _windows(x, edge, w)
    u = (seen * weight).sum(-1) + s["bias"]
    gate = torch.sigmoid(u)
    gu = grad * gate * (1 + u * (1 - gate))
    gx = (torch.cat([gu, edge], 1).unfold(1, w, 1) * weight.flip(1)).sum(-1)
    form = s["x"].dtype
    return [(u * gate).to(form), gx.to(form), (seen * gu[..., None]).sum((0, 1)), gu.sum((0, 1))]


def _plain_conv_prompt(s):
    form, w = s["x"].dtype, s["weight"].shape[1]
    u = (_windows(s["x"].float(), s["window"].float(), w) * s["weight"]).sum(-1) + s["bias"]
    y = torch.where(_valid(s), u * torch.sigmoid(u), torch.zeros_like(u)).to(form)
    rows = torch.cat([s["window"], s["x"]], 1)
    last = s["lengths"].long() if "lengths" in s else torch.full((rows.shape[0],), s["x"].shape[1], device=rows.device)
    at = last[:, None] + torch.arange(w - 1, device=rows.device)
    return [y, torch.gather(rows, 1, at[..., None].expand(-1, -1, rows.shape[2]))]


def _recurrence(a, b):
    """All h[t] = a[t] h[t-1] + b[t] (h[-1] = 0) along axis 1, in log2(T) doublings; a and b are overwritten."""
    span = 1
    while span < b.shape[1]:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _scan_terms(s):
    """delta, a = exp(delta A) and delta x in 32 bits; the rows past a sequence's length leave the state alone."""
    x, raw, keep = s["x"].float(), s["dt"].float() + s["dt_bias"], _valid(s)
    delta = torch.where(keep, _softplus(raw), torch.zeros_like(raw))
    return x, raw, delta, torch.exp(delta[..., None] * s["A"]), keep


def _plain_scan_prompt(s):
    x, _, delta, a, keep = _scan_terms(s)
    fed = (delta * x)[..., None] * s["B"].float()[:, :, None]
    fed[:, 0] += a[:, 0] * s["state"]
    h = _recurrence(a, fed)
    y = (h * s["C"].float()[:, :, None]).sum(-1) + s["D"] * x
    z = s["z"].float()
    out = torch.where(keep, y * z * torch.sigmoid(z), torch.zeros_like(y))
    return [out.to(s["x"].dtype), h[:, -1].contiguous()]


def _plain_scan_train(s):
    form = s["x"].dtype
    x, raw, delta, a, _ = _scan_terms(s)
    bm, cm, z, grad = s["B"].float(), s["C"].float(), s["z"].float(), s["grad"].float()
    h = _recurrence(a, (delta * x)[..., None] * bm[:, :, None])
    y = (h * cm[:, :, None]).sum(-1) + s["D"] * x
    gate = torch.sigmoid(z)
    out, gy = y * z * gate, grad * z * gate
    gz = grad * y * gate * (1 + z * (1 - gate))
    gc = (h * gy[..., None]).sum(2)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * a
    del h
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    del a
    g = _recurrence(later, (gy[..., None] * cm[:, :, None]).flip(1)).flip(1)
    del later
    gb = (g * (delta * x)[..., None]).sum(2)
    along = (g * bm[:, :, None]).sum(-1)
    held = g * before
    del g, before
    gdelta = x * along + (held * s["A"]).sum(-1)
    ga = (held * delta[..., None]).sum((0, 1))
    gdt = gdelta * torch.sigmoid(raw)
    gx = delta * along + s["D"] * gy
    gd, gbias = (gy * x).sum((0, 1)), gdt.sum((0, 1))
    return [out.to(form), gx.to(form), gdt.to(form), ga, gb.to(form), gc.to(form), gd, gz.to(form), gbias]


def _plain_step(s):
    form = s["x"].dtype
    rows = torch.cat([s["window"], s["x"][:, None]], 1)
    v = (rows.float() * s["weight"].t()).sum(1) + s["bias"]
    s["window"].copy_(rows[:, 1:])
    x = s["u"].float()
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    s["state"].copy_(torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * x)[..., None] * s["B"].float()[:, None])
    y = (s["state"] * s["C"].float()[:, None]).sum(-1) + s["D"] * x
    z = s["z"].float()
    return [(v * torch.sigmoid(v)).to(form), (y * z * torch.sigmoid(z)).to(form), s["window"], s["state"]]


def _plain_norm_train(s):
    x, grad, form = s["x"].float(), s["grad"].float(), s["x"].dtype
    off = x - x.mean(-1, keepdim=True)
    scale = torch.rsqrt((off * off).mean(-1, keepdim=True) + 1e-5)
    hat = off * scale
    gh = grad * s["weight"]
    gx = scale * (gh - gh.mean(-1, keepdim=True) - hat * (gh * hat).mean(-1, keepdim=True))
    return [(hat * s["weight"] + s["bias"]).to(form), gx.to(form), (grad * hat).sum(0), grad.sum(0)]


def _plain_matvec(s):
    k, g = s["case"]["k"], s["case"]["g"]
    q = torch.stack([s["packed"] & 15, s["packed"] >> 4], -1).flatten(1)[:, :k].float()
    group = torch.arange(k, device=q.device) // g
    weight = (q - s["zeros"].float()[:, group]) * s["scales"].float()[:, group]
    return (s["x"].float() @ weight.t()).to(s["x"].dtype)


_PLAIN = {
    "conv_train": _plain_conv_train, "conv_prompt": _plain_conv_prompt, "scan_train": _plain_scan_train, "scan_prompt": _plain_scan_prompt,
    "step": _plain_step, "norm_train": _plain_norm_train, "matvec": _plain_matvec,
}  # fmt: skip


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    with torch.no_grad():
        s = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
        return _EXACT[case["kind"]](case, s)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _silu_slope(v):
    return (1 + torch.exp(-v) * (1 + v)) / (1 + torch.exp(-v)) ** 2


def _delta(v):
    return torch.where(v > 30, v, torch.log1p(torch.exp(torch.clamp(v, max=30))))


def _exact_taps(s, front):
    """The convolution before its activation, one tap after the other."""
    rows, t, w = torch.cat([front, s["x"]], 1), s["x"].shape[1], s["weight"].shape[1]
    u = s["bias"].expand_as(s["x"]).clone()
    for j in range(w):
        u += s["weight"][:, j] * rows[:, j : j + t]
    return u, rows


def _exact_conv_train(case, s):
    w = case["w"]
    b, t, c = s["x"].shape
    u, rows = _exact_taps(s, s["x"].new_zeros(b, w - 1, c))
    gu = s["grad"] * _silu_slope(u)
    grows = torch.zeros_like(rows)
    gw = torch.zeros_like(s["weight"])
    for j in range(w):
        grows[:, j : j + t] += s["weight"][:, j] * gu
        gw[:, j] = torch.einsum("btc,btc->c", gu, rows[:, j : j + t])
    return [_silu(u), grows[:, w - 1 :], gw, gu.sum(0).sum(0)]


def _exact_conv_prompt(case, s):
    u, rows = _exact_taps(s, s["window"])
    y, kept = _silu(u), []
    for i in range(case["b"]):
        n = int(s["lengths"][i]) if "lengths" in s else case["t"]
        y[i, n:] = 0
        kept.append(rows[i, n : n + case["w"] - 1])
    return [y, torch.stack(kept)]


def _exact_forward(case, s, h, keep_all):
    """The recurrence token by token: y before the gate, the last state, and all states when they are asked for."""
    delta = _delta(s["dt"] + s["dt_bias"])
    ys, hs = [], []
    for t in range(case["t"]):
        new = torch.exp(delta[:, t, :, None] * s["A"]) * h + delta[:, t, :, None] * s["B"][:, t, None] * s["x"][:, t, :, None]
        if "lengths" in s:
            new = torch.where((t < s["lengths"])[:, None, None], new, h)
        h = new
        ys.append(torch.einsum("bcn,bn->bc", h, s["C"][:, t]) + s["D"] * s["x"][:, t])
        if keep_all:
            hs.append(h)
    return torch.stack(ys, 1), h, hs


def _exact_scan_prompt(case, s):
    y, h, _ = _exact_forward(case, s, s["state"], False)
    out = y * _silu(s["z"])
    if "lengths" in s:
        for i in range(case["b"]):
            out[i, int(s["lengths"][i]) :] = 0
    return [out, h]


def _exact_scan_train(case, s):
    b, t, c, n = case["b"], case["t"], case["c"], case["n"]
    if b * t * c * n > 450_000_000:
        return None
    zero = s["x"].new_zeros(b, c, n)
    y, _, hs = _exact_forward(case, s, zero, True)
    raw = s["dt"] + s["dt_bias"]
    delta, gy = _delta(raw), s["grad"] * _silu(s["z"])
    ga, g = torch.zeros_like(s["A"]), zero
    gx, gdelta = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    gb, gc = torch.empty_like(s["B"]), torch.empty_like(s["C"])
    for i in range(t - 1, -1, -1):
        d, x = delta[:, i, :, None], s["x"][:, i, :, None]
        g = g + gy[:, i, :, None] * s["C"][:, i, None]
        gc[:, i] = torch.einsum("bc,bcn->bn", gy[:, i], hs[i])
        gb[:, i] = (g * d * x).sum(1)
        fed = (g * s["B"][:, i, None]).sum(2)
        decay = torch.exp(d * s["A"])
        held = g * decay * (hs[i - 1] if i else zero)
        gx[:, i] = delta[:, i] * fed + s["D"] * gy[:, i]
        gdelta[:, i] = s["x"][:, i] * fed + (held * s["A"]).sum(2)
        ga += (held * d).sum(0)
        g = g * decay
        hs.pop()
    gdt = gdelta / (1 + torch.exp(-raw))
    gz = s["grad"] * y * _silu_slope(s["z"])
    return [y * _silu(s["z"]), gx, gdt, ga, gb, gc, torch.einsum("btc,btc->c", gy, s["x"]), gz, gdt.sum(0).sum(0)]


def _exact_step(case, s):
    v = s["bias"] + s["weight"][:, -1] * s["x"]
    for j in range(case["w"] - 1):
        v = v + s["weight"][:, j] * s["window"][:, j]
    x = s["u"]
    d = _delta(s["dt"] + s["dt_bias"])[..., None]
    h = torch.exp(d * s["A"]) * s["state"] + d * x[..., None] * s["B"][:, None]
    y = torch.einsum("bcn,bn->bc", h, s["C"]) + s["D"] * x
    return [_silu(v), y * _silu(s["z"]), torch.cat([s["window"][:, 1:], s["x"][:, None]], 1), h]


def _exact_norm_train(case, s):
    x, c = s["x"], case["c"]
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    std = torch.sqrt(var + 1e-5)
    y = (x - mean) / std
    gy = s["grad"] * s["weight"]
    inner = torch.einsum("rc,rc->r", gy, y)[:, None] / c
    gx = (gy - gy.sum(-1, keepdim=True) / c - y * inner) / std
    return [y * s["weight"] + s["bias"], gx, torch.einsum("rc,rc->c", s["grad"], y), s["grad"].sum(0)]


def _exact_matvec(case, s):
    k, g, n = case["k"], case["g"], case["n"]
    y = s["x"].new_zeros(case["m"], n)
    for i in range(-(-k // g)):
        lo, hi = i * g, min(k, i * g + g)
        packed = s["packed"][:, lo // 2 : (hi + 1) // 2]
        q = torch.empty((n, 2 * packed.shape[1]), dtype=torch.float64, device=y.device)
        q[:, 0::2], q[:, 1::2] = packed % 16, packed // 16
        part = s["x"][:, lo:hi] @ (q[:, : hi - lo] - s["zeros"][:, i : i + 1]).t()
        y += part * s["scales"][:, i]
    return y


_EXACT = {
    "conv_train": _exact_conv_train, "conv_prompt": _exact_conv_prompt, "scan_train": _exact_scan_train, "scan_prompt": _exact_scan_prompt,
    "step": _exact_step, "norm_train": _exact_norm_train, "matvec": _exact_matvec,
}  # fmt: skip
