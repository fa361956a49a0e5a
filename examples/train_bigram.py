"""Trains a small language model whose every operator is one of hc.gfx950's.

The model predicts a token from the one before it: the token's embedding, a
layer norm, and a linear head that shares the embedding's table.  A step is

    embedding -> layer_norm -> linear_cross_entropy_grad
              -> layer_norm_grad -> embedding_grad -> update

with the parameters held in float32 and rounded to bfloat16 for the step.  The
table has two gradients, the head's and the embedding's.  The text is synthetic:
each token is followed by one fixed token, except that one in ten is random
(an entropy of about 0.1 log(vocabulary) + 0.33).

    python examples/train_bigram.py [--steps 200] [--tokens 8192] [--vocab 4096] [--width 512]
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "5_amd"))

import hc.gfx950 as g  # noqa: E402

BF16 = torch.bfloat16
PAD = -100  # the target of a position without a next token
RANDOM = 0.1  # of the text's tokens


class Bigram:
    """The parameters in float32, their bfloat16 forms, and Adam's moments."""

    def __init__(self, vocab: int, width: int, device: str, seed: int = 0) -> None:
        gen = torch.Generator(device=device).manual_seed(seed)
        self.scale = math.sqrt(width)
        table = torch.randn((vocab, width), generator=gen, device=device) / math.sqrt(width)
        self.params = [table, torch.ones((width,), device=device), torch.zeros((width,), device=device)]
        self.moments = [(torch.zeros_like(p), torch.zeros_like(p)) for p in self.params]
        self.steps = 0

    def loss_and_grads(self, tokens: torch.Tensor, targets: torch.Tensor) -> tuple[torch.Tensor, list[torch.Tensor]]:
        table, weight, bias = (p.to(BF16) for p in self.params)
        e = g.embedding(tokens, table, scale=self.scale)
        h, mean, rstd = g.layer_norm(e, weight, bias)
        loss, dh, dtable = g.linear_cross_entropy_grad(h, table, targets, ignore_index=PAD)
        de, dweight, dbias = g.layer_norm_grad(dh, e, mean, rstd, weight, param_dtype=torch.float32)
        through = g.embedding_grad(de, tokens, table.shape[0], scale=self.scale, dtype=torch.float32)
        return loss, [through.add_(dtable), dweight, dbias]

    def losses(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        """Every position's loss, without gradients."""
        table, weight, bias = (p.to(BF16) for p in self.params)
        h, _, _ = g.layer_norm(g.embedding(tokens, table, scale=self.scale), weight, bias)
        return g.linear_cross_entropy(h, table, targets, ignore_index=PAD)[0]

    def step(self, tokens: torch.Tensor, targets: torch.Tensor, rate: float) -> torch.Tensor:
        loss, grads = self.loss_and_grads(tokens, targets)
        self.steps += 1
        for p, d, (m, v) in zip(self.params, grads, self.moments):
            m.lerp_(d, 0.1)
            v.lerp_(d * d, 0.01)
            p.sub_(rate * (m / (1 - 0.9**self.steps)) / ((v / (1 - 0.99**self.steps)).sqrt() + 1e-8))
        return loss


def text(rows: int, length: int, follows: torch.Tensor, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens, targets), both rows x length; the last position has no target."""
    vocab = follows.shape[0]
    shape = (rows, length)
    noise = torch.randint(0, vocab, shape, generator=gen, device=follows.device)
    random = torch.rand(shape, generator=gen, device=follows.device) < RANDOM
    tokens = noise.clone()
    for i in range(1, length):
        tokens[:, i] = torch.where(random[:, i], noise[:, i], follows[tokens[:, i - 1]])
    targets = torch.full_like(tokens, PAD)
    targets[:, :-1] = tokens[:, 1:]
    return tokens, targets


def train(steps: int, tokens: int, vocab: int, width: int, rate: float = 0.01, device: str = "cuda:0",
          report: int = 20) -> tuple[float, float]:
    """(the first step's loss, the loss on a text that was not trained on)."""
    gen = torch.Generator(device=device).manual_seed(1)
    follows = torch.randperm(vocab, generator=gen, device=device)
    model = Bigram(vocab, width, device)
    length = min(64, tokens)
    first = math.nan
    for i in range(steps):
        loss = model.step(*text(max(1, tokens // length), length, follows, gen), rate)
        if i == 0:
            first = float(loss)
        if report and i % report == 0:
            print(f"step {i}: loss {float(loss):.4f}", flush=True)
    seen, targets = text(max(1, tokens // length), length, follows, gen)
    held = model.losses(seen, targets)
    return first, float(held.sum() / (targets != PAD).sum())


def main() -> None:
    p = argparse.ArgumentParser(description="Train a bigram model with hc.gfx950's operators.")
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--tokens", type=int, default=8192, help="tokens per step")
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--width", type=int, default=512)
    a = p.parse_args()
    first, held = train(a.steps, a.tokens, a.vocab, a.width)
    print(f"loss at the start {first:.4f}, on new text {held:.4f} (log vocabulary {math.log(a.vocab):.4f})")


if __name__ == "__main__":
    main()
