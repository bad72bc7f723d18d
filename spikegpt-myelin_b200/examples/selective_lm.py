"""Train a small selective state-space model, then generate with 4-bit projections.

    python spikegpt-myelin_b200/examples/selective_lm.py [--steps 500]

The task is synthetic: sequences over 64 symbols that repeat with a period of 3 to 8
tokens, so the model has to hold the period's tokens in its state. Training runs under
bfloat16 autocast through causal_conv, selective_scan and layer_norm and their
gradients; generation reads prompts of several lengths in one batch and then goes
token by token through the operators' single-token steps, with the projections'
weights in 4 bits, replayed from a CUDA graph.
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from spikegpt_b200.selective_model import SelectiveConfig, SelectiveLM  # noqa: E402


def periodic(batch: int, length: int, symbols: int, rng: torch.Generator) -> torch.Tensor:
    rows = []
    for _ in range(batch):
        period = int(torch.randint(3, 9, (1,), generator=rng))
        unit = torch.randint(0, symbols, (period,), generator=rng)
        rows.append(unit.repeat(length // period + 1)[:length])
    return torch.stack(rows)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=500)
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--length", type=int, default=128)
    args = ap.parse_args()
    rng = torch.Generator().manual_seed(0)
    torch.manual_seed(0)
    config = SelectiveConfig(vocab_size=64, n_layer=2, n_embd=128)
    model = SelectiveLM(config).cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.01, fused=True)
    for step in range(args.steps):
        ids = periodic(args.batch, args.length + 1, config.vocab_size, rng).cuda()
        with torch.autocast("cuda", torch.bfloat16):
            loss = model(ids[:, :-1], ids[:, 1:])
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if step % 100 == 0 or step == args.steps - 1:
            print(f"step {step}: loss {loss.item():.3f}", flush=True)

    # prompts of several lengths, continued with 4-bit projections
    model = model.to(torch.bfloat16).quantize_(group_size=64)
    text = periodic(4, 96, config.vocab_size, rng).cuda()
    lengths = torch.tensor([24, 40, 33, 64], device="cuda")
    logits, states = model.prefill(text[:, :64], lengths)
    token = logits.argmax(-1)
    model.step(token, [type(s)(s.window.clone(), s.state.clone()) for s in states])  # warm-up on copies
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        following = model.step(token, states).argmax(-1)
    said = [token.clone()]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(31):
        graph.replay()
        token.copy_(following)
        said.append(token.clone())
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / 31
    said = torch.stack(said, 1)
    want = torch.stack([text[i, n : n + 32] for i, n in enumerate(lengths.tolist())])
    right = (said == want).float().mean().item()
    print(f"generated 32 tokens after each of 4 prompts: {100 * right:.0f} % as the period has them, "
          f"{1e6 * took:.0f} us a token")


if __name__ == "__main__":
    main()
