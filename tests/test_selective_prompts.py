"""Prompts of the selective model at the ends of their lengths: none, and more than
there are rows. The host side on the CPU; the model on the GPU."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from spikegpt_b200 import selective_model
from spikegpt_b200.selective_model import SelectiveConfig, SelectiveLM, SelectiveState

CONFIG = SelectiveConfig(vocab_size=50, n_layer=2, n_embd=48, inner=80, n_state=16, taps=4, dt_rank=5)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_logits_are_of_the_last_token_or_of_zeros(monkeypatch, kind):
    """The blocks stand aside, so the logits show which row of the embedding they are of. A
    length of 0 must not read the padding, one past T no row that does not exist."""
    monkeypatch.setattr(selective_model, "layer_norm", lambda x, w, b: F.layer_norm(x, x.shape[-1:], w, b))
    monkeypatch.setattr(selective_model.SelectiveBlock, "forward",
                        lambda self, x, lengths=None, return_state=False: (x, SelectiveState(x, x)))
    torch.manual_seed(0)
    model = SelectiveLM(CONFIG)
    ids = torch.randint(0, 50, (5, 7), generator=torch.Generator().manual_seed(1))
    lengths = torch.tensor([7, 0, 3, 9, -2], dtype=kind)
    logits, _ = model.prefill(ids, lengths)
    stream = model.embedding(ids)
    want = torch.stack([stream[0, 6], torch.zeros(48), stream[2, 2], stream[3, 6], torch.zeros(48)])
    want = model.head(F.layer_norm(want, (48,), model.norm_weight, model.norm_bias))
    torch.testing.assert_close(logits, want)
    whole, _ = model.prefill(ids)
    torch.testing.assert_close(whole, model.head(F.layer_norm(stream[:, -1], (48,))))
    for none in (None, torch.zeros(5, dtype=kind)):
        logits, _ = model.prefill(ids[:, :0], none)
        torch.testing.assert_close(logits, model.head(model.norm_bias).expand(5, -1))


@pytest.mark.gpu
def test_a_prompt_of_no_tokens_reads_no_padding(cuda):
    torch.manual_seed(1)
    model = SelectiveLM(CONFIG).to(cuda)
    ids = torch.randint(0, 50, (4, 25), generator=torch.Generator().manual_seed(3)).to(cuda)
    lengths = torch.tensor([25, 0, 13, 40], device=cuda)
    logits, states = model.prefill(ids, lengths)
    others = ids.clone()
    others[1] = (ids[1] + 7) % 50
    again, _ = model.prefill(others, lengths)
    assert torch.equal(logits, again) and torch.isfinite(logits).all()
    assert all((s.state[1] == 0).all() and (s.window[1] == 0).all() for s in states)
    torch.testing.assert_close(logits[1], model.head(model.norm_bias))
    full, _ = model.prefill(ids[3:], None)
    torch.testing.assert_close(logits[3:], full, rtol=1e-4, atol=1e-5)
    empty, none = model.prefill(ids[:, :0])
    torch.testing.assert_close(empty, model.head(model.norm_bias).expand(4, -1))
    # a sequence that has read nothing goes on as one that starts with its next token
    token = ids[:, 0]
    torch.testing.assert_close(model.step(token, none), model.prefill(ids[:, :1])[0], rtol=1e-4, atol=1e-5)


def test_generate_gives_as_many_tokens_as_it_is_asked_for(monkeypatch):
    model = SelectiveLM(CONFIG)
    logits = torch.arange(100.0).view(2, 50)
    monkeypatch.setattr(model, "prefill", lambda ids, lengths=None: (logits, []))
    monkeypatch.setattr(model, "step", lambda tokens, states: logits)
    ids = torch.zeros(2, 4, dtype=torch.int32)
    for count in (0, 1, 2, 5):
        out = model.generate(ids, count)
        assert out.shape == (2, count) and out.dtype == torch.int64 and (out == 49).all()
    with pytest.raises(ValueError):
        model.generate(ids, -1)
