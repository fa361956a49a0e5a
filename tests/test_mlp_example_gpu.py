"""The example of 8-bit linear layers: its gradients against autograd in 64
bits, and that it runs."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "train_mlp.py")
    spec = importlib.util.spec_from_file_location("train_mlp", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("vocab,width,rows,length", [(300, 72, 9, 31), (500, 128, 3, 50)])
def test_gradients(vocab, width, rows, length):
    """One step against autograd of the same model in 64 bits, by norms.  A
    quantised operand errs by at most u / sqrt(3) of its norm, u = 2^-4 (e4m3)
    or 2^-3 (e5m2): 0.036 and 0.072.  A gradient passes at most three products
    each way (a block's two layers and its weight's own), whose operands are e4m3
    in the forward pass (two each) and one of them e5m2 in the backward pass, and
    the square doubles what reaches it: 3 * 2 * 0.036 * 2 + 3 * (0.036 + 0.072) =
    0.76 of the norm at the worst, where all errors have one direction.  They are
    independent: the root of the sum of their squares is sqrt(24 + 3) * 0.036 +
    ... < 0.23, and 0.4 leaves a factor for single parameters of few values."""
    ex = _example()
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    model = ex.Model(vocab, width, 1, "cuda:0")
    tokens, targets = ex.text(rows, length, torch.randperm(vocab, generator=gen, device="cuda:0"), gen)
    loss, grads = model.loss_and_grads(tokens, targets)
    p = [q.double().requires_grad_() for q in model.params]

    def norm(h, w):
        return h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    h = p[0][tokens] * model.scale
    h = h + (norm(h, p[1]) @ p[2].t()).relu().square() @ p[3].t()
    want = torch.nn.functional.cross_entropy((norm(h, p[4]) @ p[0].t()).flatten(0, 1), targets.flatten(),
                                             ignore_index=ex.PAD)
    want.backward()
    assert abs(float(loss) - float(want.detach())) <= 0.1 * float(want.detach())
    for got, q in zip(grads, p):
        assert got.dtype == torch.float32 and got.shape == q.shape
        assert float((got.double() - q.grad).norm()) <= 0.4 * float(q.grad.norm())


def test_runs():
    losses = _example().train(steps=4, tokens=512, vocab=256, width=64, layers=2, report=0)
    assert len(losses) == 4 and all(math.isfinite(v) for v in losses)
