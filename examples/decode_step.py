"""Speculative decoding with a coded decoder: every step verifies a batch's drafted tokens.

Between the coded projections (dense.Dense, experts) run the operators around them:

    embed -> norm -> [ q/k/v + adapters -> mixer -> o + adapters -> stream + norm -> experts -> stream + norm ] x layers
          -> coded LM head -> verification of the drafted tokens

norms.BlockNorm carries the residual stream and gives the next block its input in one pass (after the experts with their two
outputs), adapters.Adapters adds each request's low-rank adapter beside the shared coded weights, speculative.verify turns
the head's logits into the step's tokens. The weights are random, the mixer is an elementwise stand-in for attention, and
the drafter guesses the target's own likeliest tokens part of the time; what is real is the path.

    python examples/decode_step.py [--layers 4 --hidden 2048 --vocab 32000 --requests 6 --drafts 3 --steps 8]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from vllm_espalier_b200 import adapters, dense, experts, norms, speculative  # noqa: E402


class Coded:
    """A random coded matrix: uniform trellis states, +-1 input signs, small output scales."""

    def __init__(self, kin: int, n: int, bits: int, grid: int, gen: torch.Generator):
        dev = gen.device
        self.trellis = torch.randint(-32768, 32768, (kin // 16, n // 16, 16 * bits), dtype=torch.int16, device=dev,
                                     generator=gen)
        self.suh = (torch.randint(0, 2, (kin,), device=dev, generator=gen) * 2 - 1).half()
        self.svh = ((torch.rand(n, device=dev, generator=gen) + 0.5) / 64).half()
        self.K, self.cb, self.in_features, self.out_features = bits, grid, kin, n


class Decoder:
    def __init__(self, dev, layers: int = 2, hidden: int = 512, kv: int = 128, inter: int = 256, n_experts: int = 8,
                 top_k: int = 2, vocab: int = 4096, slots: int = 4, rank: int = 16, rows: int = 32, seed: int = 0):
        gen = torch.Generator(device=dev).manual_seed(seed)
        q = 2 * hidden
        self.hidden, self.q, self.kv, self.vocab, self.top_k, self.rows = hidden, q, kv, vocab, top_k, rows

        def normal(*shape, std=1.0, mean=0.0):
            return (torch.randn(*shape, device=dev, generator=gen) * std + mean).to(torch.bfloat16)

        def adapter(k, widths):
            return adapters.Adapters(normal(slots, len(widths), rank, k, std=k ** -0.5),
                                     normal(slots, sum(widths), rank, std=rank ** -0.5), widths,
                                     scales=torch.rand(slots, device=dev, generator=gen))
        self.embed = normal(vocab, hidden)
        self.layers = []
        for _ in range(layers):
            expert = [tuple(Coded(a, b, 3, 3, gen) for a, b in ((hidden, inter), (hidden, inter), (inter, hidden)))
                      for _ in range(n_experts)]
            shared = tuple(Coded(a, b, 4, 4, gen) for a, b in ((hidden, inter), (hidden, inter), (inter, hidden)))
            self.layers.append({
                "qkv": dense.Dense([Coded(hidden, n, 4, 3, gen) for n in (q, kv, kv)]),
                "o": dense.Dense([Coded(q, hidden, 4, 3, gen)]),
                "qkv_adapters": adapter(hidden, [q, kv, kv]), "o_adapters": adapter(q, [hidden]),
                "moe": experts.prepare(expert, shared, normal(hidden, std=hidden ** -0.5)),
                "router": normal(n_experts, hidden, std=hidden ** -0.5),
            })
        weights = [normal(hidden, std=0.05, mean=1.0) for _ in range(2 * layers + 1)]
        # the norm before each block and, after the last, before the head; each but the first also adds to the stream
        self.first = norms.BlockNorm(hidden, pre=weights[0])
        self.between = [norms.BlockNorm(hidden, pre=w, block_scale=0.5) for w in weights[1:]]
        self.head = dense.Dense([Coded(hidden, vocab, 6, 0, gen)])
        self.scratch = experts.scratch(self.layers[0]["moe"], rows, top_k + 1, dev)

    def mixer(self, qkv: torch.Tensor) -> torch.Tensor:
        q, k, v = qkv.float().split([self.q, self.kv, self.kv], dim=1)
        times = self.q // self.kv
        return (torch.tanh(q) * torch.sigmoid(k.repeat(1, times)) + 0.5 * v.repeat(1, times)).to(qkv.dtype)

    def logits(self, tokens: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """tokens int64 [rows <= 32], ids int32 [rows] (the adapter of each row, -1: none) -> logits [rows, vocab]."""
        stream, h = self.first(self.embed[tokens])
        for i, layer in enumerate(self.layers):
            qkv = layer["qkv"].forward(h)
            layer["qkv_adapters"].forward(h, qkv, ids, out=qkv)
            core = self.mixer(qkv)
            block = layer["o"].forward(core)
            layer["o_adapters"].forward(core, block, ids, out=block)
            stream, h = self.between[2 * i](block, stream)
            experts.route(h, layer["router"], self.top_k, layer["moe"], self.scratch)
            routed, shared = experts.routed2(h, None, None, layer["moe"], self.scratch, k=self.top_k)
            stream, h = self.between[2 * i + 1](routed, stream, x2=shared)
        return self.head.forward(h)


class Batch:
    """The requests of a decode loop, each with its adapter and temperature; one call of step() a decode step."""

    def __init__(self, model: Decoder, requests: int, drafts: int, seed: int = 1):
        dev = model.embed.device
        if requests * (drafts + 1) > model.rows:
            raise ValueError(f"{requests} requests of {drafts} drafted tokens are more than {model.rows} rows")
        self.model, self.B, self.k = model, requests, drafts
        self.gen = torch.Generator(device=dev).manual_seed(seed)
        self.last = torch.randint(0, model.vocab, (requests,), device=dev, generator=self.gen)
        ids = torch.arange(requests, device=dev, dtype=torch.int32) % 5 - 1         # one request in five without one
        self.ids = ids.repeat_interleave(drafts + 1)
        self.starts = torch.arange(requests + 1, device=dev, dtype=torch.int32) * drafts
        self.temperature = torch.where(torch.arange(requests, device=dev) % 3 == 2, 0.0, 0.8)

    def draft(self) -> torch.Tensor:
        """[B, k] guesses: the model's likeliest continuation of the last token, half of them spoiled. (A real drafter is a
        small model; this one asks the target itself.)"""
        token, out = self.last, []
        for _ in range(self.k):
            token = self.model.logits(token, self.ids[::self.k + 1].contiguous()).argmax(1)
            spoiled = torch.rand(self.B, device=token.device, generator=self.gen) < 0.3
            token = torch.where(spoiled, (token + 1) % self.model.vocab, token)
            out.append(token)
        return torch.stack(out, 1) if out else self.last.new_empty((self.B, 0))

    def step(self):
        """One step: (tokens int32 [B, k + 1] with -1 after each request's own, accepted int32 [B], probs)."""
        drafted = self.draft()
        rows = torch.cat([self.last[:, None], drafted], 1).reshape(-1)
        logits = self.model.logits(rows, self.ids)
        dev = logits.device
        noise = torch.empty((self.B, self.model.vocab), device=dev).exponential_(generator=self.gen).clamp_(min=1e-30)
        tokens, accepted, probs = speculative.verify(
            logits[:, :self.model.vocab], self.starts, drafted.reshape(-1).to(torch.int32),
            torch.rand(self.B * self.k, device=dev, generator=self.gen), noise, self.k, temperature=self.temperature)
        self.last = tokens.gather(1, accepted[:, None].long())[:, 0].long()
        return tokens, accepted, probs


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("layers", 4), ("hidden", 2048), ("vocab", 32000), ("requests", 6), ("drafts", 3), ("steps", 8)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    model = Decoder(torch.device("cuda:0"), layers=a.layers, hidden=a.hidden, vocab=a.vocab)
    batch = Batch(model, a.requests, a.drafts)
    emitted = 0
    for i in range(a.steps):
        tokens, accepted, _ = batch.step()
        emitted += int((tokens >= 0).sum())
        print(f"step {i}: accepted {accepted.tolist()} of {a.drafts}, tokens {tokens.tolist()}")
    print(f"{emitted} tokens in {a.steps} steps of {a.requests} requests "
          f"({emitted / (a.steps * a.requests):.2f} a request and step)")


if __name__ == "__main__":
    main()
