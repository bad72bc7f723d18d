"""GPU tests of the selective model: its forward and gradients against the same model
in plain 64-bit torch operations, prompts and single tokens against the whole
sequence, right-padded prompts, 4-bit projections, a CUDA graph of the step, and
training."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F
from _mixertest import conv_ref, scan_ref

from spikegpt_b200.selective_model import Q4Linear, SelectiveConfig, SelectiveLM

pytestmark = pytest.mark.gpu

CONFIG = SelectiveConfig(vocab_size=50, n_layer=2, n_embd=48, inner=80, n_state=16, taps=4, dt_rank=5)


def _model(device, dtype=torch.float32, config=CONFIG):
    torch.manual_seed(1)
    return SelectiveLM(config).to(device=device, dtype=dtype)


def _plain(model, ids):
    """The model's logits in its parameters' own (64-bit) type, without its operators."""
    x = model.embedding(ids)
    c = (x.shape[-1],)
    for b in model.blocks:
        u, z = b.in_proj(F.layer_norm(x, c, b.norm_weight, b.norm_bias)).chunk(2, -1)
        u, _ = conv_ref(u, b.conv_weight, b.conv_bias)
        dt, B, C = b._split(u)
        y, _ = scan_ref(u, dt, -torch.exp(b.A_log), B, C, b.D, z, b.dt_bias)
        x = x + b.out_proj(y)
    return model.head(F.layer_norm(x, c, model.norm_weight, model.norm_bias))


def _ids(b, t, device, seed=0):
    return torch.randint(0, CONFIG.vocab_size, (b, t), generator=torch.Generator().manual_seed(seed)).to(device)


def test_forward_and_gradients_match_plain_operations(cuda):
    """Two layers of a few hundred float32 roundings each: 1e-4 of the largest value."""
    model = _model(cuda)
    wide = copy.deepcopy(model).double()
    ids = _ids(3, 41, cuda)
    logits, ref = model(ids), _plain(wide, ids)
    assert float((logits.double() - ref).detach().abs().max()) <= 1e-4 * float(ref.detach().abs().max())
    model(ids[:, :-1], ids[:, 1:]).backward()
    F.cross_entropy(_plain(wide, ids[:, :-1]).reshape(-1, 50), ids[:, 1:].reshape(-1)).backward()
    for (name, p), q in zip(model.named_parameters(), wide.parameters()):
        scale = float(q.grad.abs().max())
        assert scale > 0 and float((p.grad.double() - q.grad).abs().max()) <= 2e-4 * scale, name


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
def test_prompt_and_steps_follow_the_sequence(cuda, dtype, tol):
    """bfloat16: the residual stream and the projections round to 2^-9 in either form, in
    different places; a handful of such roundings of the logits' scale."""
    model = _model(cuda, dtype)
    ids = _ids(2, 30, cuda, seed=2)
    with torch.no_grad():
        whole = model(ids).float()
        logits, states = model.prefill(ids[:, :19])
        scale = float(whole.abs().max())
        assert float((logits.float() - whole[:, 18]).abs().max()) <= tol * scale
        for t in range(19, 30):
            logits = model.step(ids[:, t], states)
            assert float((logits.float() - whole[:, t]).abs().max()) <= tol * scale, t


def test_right_padded_prompts(cuda):
    model = _model(cuda)
    ids = _ids(4, 25, cuda, seed=3)
    lengths = torch.tensor([25, 1, 13, 4], device=cuda)
    inputs = []  # what each block's convolution read: a window is those values, to the bit
    hooks = [b.in_proj.register_forward_hook(lambda m, a, out: inputs.append(out)) for b in model.blocks]
    logits, states = model.prefill(ids, lengths)
    for hook in hooks:
        hook.remove()
    for i, n in enumerate(lengths.tolist()):
        alone, one = model.prefill(ids[i : i + 1, :n])
        torch.testing.assert_close(logits[i : i + 1], alone, rtol=1e-4, atol=1e-5)
        for s, o, read in zip(states, one, inputs):
            past = F.pad(read[i, :n, : CONFIG.inner], (0, 0, 3, 0))[-3:]
            assert torch.equal(s.window[i], past)
            torch.testing.assert_close(s.state[i : i + 1], o.state, rtol=1e-4, atol=1e-6)


def test_four_bit_projections_are_their_decoded_weights(cuda):
    model = _model(cuda).quantize_(32)
    plain = _model(cuda)
    for b, p in zip(model.blocks, plain.blocks):
        for name in ("in_proj", "x_proj", "out_proj"):
            q = getattr(b, name)
            assert isinstance(q, Q4Linear)
            getattr(p, name).weight.data.copy_(q.weight())
    plain.head.weight.data.copy_(model.head.weight())
    ids = _ids(3, 20, cuda, seed=4)
    a, sa = model.prefill(ids[:, :12])
    b, sb = plain.prefill(ids[:, :12])
    torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4)
    for t in range(12, 20):
        torch.testing.assert_close(model.step(ids[:, t], sa), plain.step(ids[:, t], sb), rtol=1e-3, atol=1e-4)


def test_step_replays_from_a_graph(cuda):
    model = _model(cuda, torch.bfloat16).quantize_(32)
    ids = _ids(2, 9, cuda, seed=5)
    want = model.generate(ids, 6)
    logits, states = model.prefill(ids)
    token = logits.argmax(-1)
    model.step(token, [type(s)(s.window.clone(), s.state.clone()) for s in states])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        following = model.step(token, states).argmax(-1)
    got = [token.clone()]
    for _ in range(5):
        graph.replay()
        token.copy_(following)
        got.append(token.clone())
    assert torch.equal(torch.stack(got, 1), want)


def test_training_under_autocast_learns(cuda):
    model = _model(cuda)
    opt = torch.optim.AdamW(model.parameters(), lr=5e-3)
    ids = _ids(8, 33, cuda, seed=6)  # a fixed batch, to be learnt by heart
    losses = []
    for _ in range(60):
        with torch.autocast("cuda", torch.bfloat16):
            loss = model(ids[:, :-1], ids[:, 1:])
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0], losses[::10]
