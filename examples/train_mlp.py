"""Trains a small language model whose layers are 8-bit linear layers.

The model predicts a token from the one before it: the token's embedding is the
residual stream, L blocks add to it, and a linear head that shares the
embedding's table reads its norm.  A block is

    rms_norm_fp8 (adds the block before's output to the residual)
      -> linear_fp8 (width -> hidden) -> square of the positive part
      -> quantize_fp8 -> linear_fp8 (hidden -> width)

A layer's gradients are two more products: with the weight quantised transposed
for its input, and of both operands quantised along the tokens for its weight, in
float32.  Parameters are float32 and are quantised or rounded to bfloat16 for the
step; the residual is float32.  The text is synthetic: each token is followed by
one fixed token, except that one in ten is random.

    python examples/train_mlp.py [--steps 200] [--tokens 8192] [--vocab 4096] [--width 512] [--layers 2]
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "5_amd"))

import hc.gfx950 as g  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
E5M2 = torch.float8_e5m2
PAD = -100  # the target of a position without a next token
RANDOM = 0.1  # of the text's tokens


class Linear:
    """The 8-bit forms of a weight (outputs x inputs) for a step, and the
    products with them."""

    def __init__(self, weight: torch.Tensor) -> None:
        self.forward_operand = g.quantize_fp8(weight, block="tile")
        self.backward_operand = g.quantize_fp8(weight, block="tile", transpose=True)

    def __call__(self, x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        return g.linear_fp8(x, scale, *self.forward_operand)

    def input_grad(self, dy: torch.Tensor) -> torch.Tensor:
        return g.linear_fp8(*g.quantize_fp8(dy, dtype=E5M2), *self.backward_operand)

    @staticmethod
    def weight_grad(dy: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        return g.linear_fp8(*g.quantize_fp8(dy, transpose=True, dtype=E5M2), *g.quantize_fp8(x, transpose=True),
                            out_dtype=F32)


class Model:
    """The parameters in float32 (table, then per block norm, up and down, then
    the last norm) and Adam's moments."""

    def __init__(self, vocab: int, width: int, layers: int, device: str, seed: int = 0) -> None:
        gen = torch.Generator(device=device).manual_seed(seed)
        hidden = 4 * width

        def normal(*shape: int) -> torch.Tensor:
            return torch.randn(shape, generator=gen, device=device) / math.sqrt(shape[-1])

        self.params = [normal(vocab, width)]
        for _ in range(layers):
            self.params += [torch.ones((width,), device=device), normal(hidden, width), normal(width, hidden)]
        self.params.append(torch.ones((width,), device=device))
        self.layers = layers
        self.scale = math.sqrt(width)
        self.moments = [(torch.zeros_like(p), torch.zeros_like(p)) for p in self.params]
        self.steps = 0

    def loss_and_grads(self, tokens: torch.Tensor, targets: torch.Tensor) -> tuple[torch.Tensor, list[torch.Tensor]]:
        table = self.params[0].to(BF16)
        out = g.embedding(tokens, table, scale=self.scale)
        residual = torch.zeros(out.shape, dtype=F32, device=out.device)
        blocks = []
        for i in range(self.layers):
            norm, up, down = (p for p in self.params[1 + 3 * i : 4 + 3 * i])
            norm, up, down = norm.to(BF16), Linear(up), Linear(down)
            q, s, residual, rstd = g.rms_norm_fp8(out, norm, residual)
            a = up(q, s)
            act = a.relu().square()
            out = down(*g.quantize_fp8(act))
            blocks.append((norm, up, down, residual, rstd, a, act))
        last = self.params[-1].to(BF16)
        h, residual, rstd = g.rms_norm(out, last, residual)

        loss, dh, dtable = g.linear_cross_entropy_grad(h, table, targets, ignore_index=PAD)
        # The gradient of a sum is one for what was added and for the residual.
        dres, dlast = g.rms_norm_grad(dh, residual, rstd, last, param_dtype=F32)
        grads = [dlast]
        for norm, up, down, held, rstd, a, act in reversed(blocks):
            dout = dres.to(BF16)
            da = down.input_grad(dout) * (2 * a.relu())
            n = g.rms_norm(held.to(BF16), norm)[0]  # (what the layer read, before its 8 bits)
            dn = up.input_grad(da)
            grads = [up.weight_grad(da, n), down.weight_grad(dout, act)] + grads
            dres, dnorm = g.rms_norm_grad(dn, held, rstd, norm, dresidual=dres, param_dtype=F32)
            grads = [dnorm] + grads
        through = g.embedding_grad(dres.to(BF16), tokens, table.shape[0], scale=self.scale, dtype=F32)
        return loss, [through.add_(dtable)] + grads

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


def train(steps: int, tokens: int, vocab: int, width: int, layers: int, rate: float = 0.003, device: str = "cuda:0",
          report: int = 20) -> list[float]:
    """The losses of the steps."""
    gen = torch.Generator(device=device).manual_seed(1)
    follows = torch.randperm(vocab, generator=gen, device=device)
    model = Model(vocab, width, layers, device)
    length = min(64, tokens)
    losses = []
    for i in range(steps):
        losses.append(model.step(*text(max(1, tokens // length), length, follows, gen), rate))
        if report and i % report == 0:
            print(f"step {i}: loss {float(losses[-1]):.4f}", flush=True)
    return [float(loss) for loss in losses]


def main() -> None:
    p = argparse.ArgumentParser(description="Train a small model of 8-bit linear layers with hc.gfx950's operators.")
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--tokens", type=int, default=8192, help="tokens per step")
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--width", type=int, default=512)
    p.add_argument("--layers", type=int, default=2)
    a = p.parse_args()
    losses = train(a.steps, a.tokens, a.vocab, a.width, a.layers)
    print(f"loss at the start {losses[0]:.4f}, at the end {losses[-1]:.4f} (log vocabulary {math.log(a.vocab):.4f})")


if __name__ == "__main__":
    main()
