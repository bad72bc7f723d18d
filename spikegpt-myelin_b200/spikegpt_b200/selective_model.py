"""A selective state-space language model on this package's operators.

Next to ``model.SpikeGPT`` (RWKV-4 time mixing; the reference's model) this is a
small model of the other recurrence: a block is

    h = layer_norm(x);  u, z = in_proj(h);  u = causal_conv(u)
    dt, B, C = x_proj(u);  dt = dt_proj(dt)
    x = x + out_proj(selective_scan(u, dt, A, B, C, D, z))

It trains (``forward``), reads prompts of several lengths in one right-padded batch
(``prefill``) and generates token by token (``step``) from the states that prefill
left, with ``quantize_`` turning the projections into 4-bit ones first if wanted.
u, z are halves of one projection and dt, B, C parts of another: the operators read
them in place. Train under ``torch.autocast("cuda", torch.bfloat16)`` or in float32;
``.to(torch.bfloat16)``, for generation, rounds A_log, D and the biases with the rest,
and the operators widen what is left of them.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from .norm import layer_norm
from .q4 import dequantize_q4, q4_linear, quantize_q4
from .selective import (
    MAX_STATES,
    MAX_TAPS,
    causal_conv,
    causal_conv_step_,
    selective_scan,
    selective_scan_step_,
)

# Tokens up to which a 4-bit projection decodes its weight on the fly; more are
# multiplied by the weight decoded once (a library matrix product).
Q4_TOKENS = 64


@dataclass
class SelectiveConfig:
    """Sizes: ``inner`` is the width of the scan (default 2 n_embd), ``dt_rank`` that of
    the step's projection (default n_embd / 16)."""

    vocab_size: int = 256
    n_layer: int = 12
    n_embd: int = 512
    inner: int = 0
    n_state: int = 16
    taps: int = 4
    dt_rank: int = 0

    def __post_init__(self) -> None:
        self.inner = self.inner or 2 * self.n_embd
        self.dt_rank = self.dt_rank or max(1, self.n_embd // 16)

    def validate(self) -> None:
        for name in ("vocab_size", "n_layer", "n_embd", "inner", "n_state", "taps", "dt_rank"):
            if getattr(self, name) <= 0:
                raise ValueError(f"{name} must be positive")
        if self.n_state > MAX_STATES or self.taps > MAX_TAPS:
            raise ValueError(f"n_state must be at most {MAX_STATES} and taps at most {MAX_TAPS}")


class Q4Linear(nn.Module):
    """A linear layer without gradient whose weight is 4-bit integers with a bfloat16
    scale and a zero point for every ``group_size`` inputs (``quantize_q4``)."""

    def __init__(self, linear: nn.Linear, group_size: int = 64) -> None:
        super().__init__()
        packed, scales, zeros = quantize_q4(linear.weight, group_size)
        self.in_features, self.out_features, self.group_size = linear.in_features, linear.out_features, group_size
        self.register_buffer("packed", packed)
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zeros)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())

    def _apply(self, fn, recurse: bool = True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != scales.dtype:  # a part of the 4-bit format, not of the model's type
            self.scales = scales.to(self.scales.device)
        return self

    def weight(self) -> Tensor:
        """The float32 weight that the packed form stands for."""
        return dequantize_q4(self.packed, self.scales, self.zeros, self.in_features, self.group_size)

    def forward(self, x: Tensor) -> Tensor:
        if x.numel() <= Q4_TOKENS * self.in_features:
            return q4_linear(x, self.packed, self.scales, self.zeros, self.bias, group_size=self.group_size)
        bias = None if self.bias is None else self.bias.to(x.dtype)
        return F.linear(x, self.weight().to(x.dtype), bias)


@dataclass
class SelectiveState:
    """What a block carries from token to token: the convolution's window
    [B, W-1, inner] and the scan's state [B, inner, N] (float32)."""

    window: Tensor
    state: Tensor


class SelectiveBlock(nn.Module):
    def __init__(self, config: SelectiveConfig) -> None:
        super().__init__()
        c, e, n, r = config.n_embd, config.inner, config.n_state, config.dt_rank
        self.config = config
        self.norm_weight = nn.Parameter(torch.ones(c))
        self.norm_bias = nn.Parameter(torch.zeros(c))
        self.in_proj = nn.Linear(c, 2 * e, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(e, config.taps).uniform_(-1, 1) / math.sqrt(config.taps))
        self.conv_bias = nn.Parameter(torch.zeros(e))
        self.x_proj = nn.Linear(e, r + 2 * n, bias=False)
        self.dt_proj = nn.Linear(r, e, bias=False)
        # steps of 0.001 to 0.1 at the start: the softplus of dt_bias
        step = torch.exp(torch.empty(e).uniform_(math.log(1e-3), math.log(1e-1)))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, n + 1, dtype=torch.float32)).repeat(e, 1))
        self.D = nn.Parameter(torch.ones(e))
        self.out_proj = nn.Linear(e, c, bias=False)

    def _split(self, u: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        r, n = self.config.dt_rank, self.config.n_state
        low = self.x_proj(u)
        return self.dt_proj(low[..., :r]), low[..., r : r + n], low[..., r + n :]

    def forward(self, x: Tensor, lengths: Tensor | None = None, return_state: bool = False):
        h = layer_norm(x, self.norm_weight, self.norm_bias)
        u, z = self.in_proj(h).chunk(2, -1)
        u = causal_conv(u, self.conv_weight, self.conv_bias, lengths=lengths, return_state=return_state)
        if return_state:
            u, window = u
        dt, B, C = self._split(u)
        y = selective_scan(u, dt, -torch.exp(self.A_log), B, C, self.D, z, self.dt_bias, lengths=lengths,
                           return_state=return_state)
        if return_state:
            y, state = y
            return x + self.out_proj(y), SelectiveState(window, state)
        return x + self.out_proj(y)

    def step(self, x: Tensor, carried: SelectiveState) -> Tensor:
        """One token, x [B, C]; ``carried`` is moved on in place."""
        h = layer_norm(x, self.norm_weight, self.norm_bias)
        u, z = self.in_proj(h).chunk(2, -1)
        u = causal_conv_step_(u, carried.window, self.conv_weight, self.conv_bias)
        dt, B, C = self._split(u)
        y = selective_scan_step_(u, dt, -torch.exp(self.A_log), B, C, carried.state, self.D, z, self.dt_bias)
        return x + self.out_proj(y)


def _last_rows(x: Tensor, lengths: Tensor | None) -> Tensor:
    """The row of x [B, T, C] at each sequence's last token, zeros where it has none; lengths
    outside 0..T count as the nearest of them, as in the operators."""
    b, t, c = x.shape
    if t == 0:
        return x.new_zeros(b, c)
    if lengths is None:
        return x[:, -1].contiguous()
    rows = x[torch.arange(b, device=x.device), lengths.long().clamp(1, t) - 1]
    return torch.where(lengths[:, None] > 0, rows, rows.new_zeros(()))


class SelectiveLM(nn.Module):
    """Embedding, ``SelectiveBlock``s, a final norm and the head. ``forward(ids,
    targets)`` returns the mean cross-entropy, ``forward(ids)`` the logits."""

    def __init__(self, config: SelectiveConfig | None = None) -> None:
        super().__init__()
        config = config or SelectiveConfig()
        config.validate()
        self.config = config
        self.embedding = nn.Embedding(config.vocab_size, config.n_embd)
        self.blocks = nn.ModuleList([SelectiveBlock(config) for _ in range(config.n_layer)])
        self.norm_weight = nn.Parameter(torch.ones(config.n_embd))
        self.norm_bias = nn.Parameter(torch.zeros(config.n_embd))
        self.head = nn.Linear(config.n_embd, config.vocab_size, bias=False)
        nn.init.normal_(self.embedding.weight, std=0.02)
        for block in self.blocks:  # the residual stream keeps its size over the layers
            block.out_proj.weight.data.div_(math.sqrt(2 * config.n_layer))

    def forward(self, ids: Tensor, targets: Tensor | None = None) -> Tensor:
        x = self.embedding(ids)
        for block in self.blocks:
            x = block(x)
        logits = self.head(layer_norm(x, self.norm_weight, self.norm_bias))
        if targets is None:
            return logits
        return F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), targets.reshape(-1))

    @torch.no_grad()
    def prefill(self, ids: Tensor, lengths: Tensor | None = None) -> tuple[Tensor, list[SelectiveState]]:
        """Logits after each sequence's last token [B, V] and the blocks' states. ``ids``
        [B, T] is padded on the right to the longest of ``lengths`` (default: all T; more
        than T counts as T). A sequence of length 0 has read nothing: its states are zeros
        and its logits those of a residual stream of zeros."""
        x = self.embedding(ids)
        states = []
        for block in self.blocks:
            x, state = block(x, lengths=lengths, return_state=True)
            states.append(state)
        return self.head(layer_norm(_last_rows(x, lengths), self.norm_weight, self.norm_bias)), states

    @torch.no_grad()
    def step(self, tokens: Tensor, states: list[SelectiveState]) -> Tensor:
        """Logits [B, V] after one more token each; ``states`` are moved on in place, so a
        CUDA graph of this call generates by replay."""
        x = self.embedding(tokens)
        for block, state in zip(self.blocks, states, strict=True):
            x = block.step(x, state)
        return self.head(layer_norm(x, self.norm_weight, self.norm_bias))

    @torch.no_grad()
    def generate(self, ids: Tensor, count: int, lengths: Tensor | None = None) -> Tensor:
        """``count`` tokens after each prompt [B, count], the most likely ones (the first
        of equals)."""
        if count < 0:
            raise ValueError(f"count must not be negative; got {count}")
        if count == 0:
            return ids.new_empty(ids.shape[0], 0, dtype=torch.long)
        logits, states = self.prefill(ids, lengths)
        out = [logits.argmax(-1)]
        for _ in range(count - 1):
            out.append(self.step(out[-1], states).argmax(-1))
        return torch.stack(out, 1)

    @torch.no_grad()
    def quantize_(self, group_size: int = 64) -> "SelectiveLM":
        """Replace the projections and the head by 4-bit ones (for generation: they have
        no gradient). The step's small projection stays as it is."""
        for block in self.blocks:
            for name in ("in_proj", "x_proj", "out_proj"):
                setattr(block, name, Q4Linear(getattr(block, name), group_size))
        self.head = Q4Linear(self.head, group_size)
        return self
