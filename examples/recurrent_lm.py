"""Train a small recurrent language model, then serve it: packed documents in training, a prefill,
and sampled decode steps in a CUDA graph on 8-bit weights.

    python examples/recurrent_lm.py [--steps 60]

The task is synthetic: documents count upwards from a random start, modulo 97.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from prime_moment_attention_b200.model import DecodeGraph, PrimeConfig, PrimeForCausalLM  # noqa: E402
from prime_moment_attention_b200.sampling import Sampler  # noqa: E402

VOCAB = 97


def documents(rows: int, length: int, gen: torch.Generator) -> torch.Tensor:
    start = torch.randint(VOCAB, (rows, 1), generator=gen, device="cuda")
    return (start + torch.arange(length, device="cuda")) % VOCAB


def main() -> float:
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    steps = ap.parse_args().steps
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    cfg = PrimeConfig(vocab_size=VOCAB, hidden_size=128, num_layers=2, num_heads=2, head_dim=64, use_recurrence=True)
    model = PrimeForCausalLM(cfg).cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for step in range(steps):
        ids = documents(16, 128, gen)
        loss = model(ids, labels=ids)["loss"]
        opt.zero_grad()
        loss.backward()
        opt.step()
        if step % 20 == 0 or step == steps - 1:
            print(f"step {step}: loss {loss.item():.3f}")

    model.eval()
    prompt = documents(8, 20, gen)
    with torch.no_grad():
        out = model(prompt, return_states=True, last_logits_only=True)
        first = out["logits"][:, -1].argmax(-1)
        graph = DecodeGraph(model, out["states"], first, sampler=Sampler(temperature=0.7, top_k=20, top_p=0.95),
                            fp8=True)
        tokens = [first]
        for _ in range(30):
            tokens.append(graph.step(torch.rand(8, generator=gen, device="cuda"))[:, 0].clone())
    got = torch.stack(tokens, 1)
    right = (got == (prompt[:, -1:] + 1 + torch.arange(31, device="cuda")) % VOCAB).float().mean().item()
    print(f"sampled continuations that count on: {right:.1%}")
    return right


if __name__ == "__main__":
    main()
