"""The bigram example: its gradients against autograd in 64 bits, and that it learns."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "train_bigram.py")
    spec = importlib.util.spec_from_file_location("train_bigram", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_gradients():
    """One step against autograd of the same model in 64 bits.  Each stage
    rounds its result to bfloat16 (2^-8 of the value), and no stage amplifies
    a relative change of its input's norm by more than a few: the gradients
    agree to 2^-4 of their norms."""
    ex = _example()
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    vocab, width = 300, 72
    model = ex.Bigram(vocab, width, "cuda:0")
    tokens, targets = ex.text(9, 31, torch.randperm(vocab, generator=gen, device="cuda:0"), gen)
    loss, grads = model.loss_and_grads(tokens, targets)
    params = [p.to(torch.bfloat16).double().requires_grad_() for p in model.params]
    e = params[0][tokens] * model.scale
    h = torch.nn.functional.layer_norm(e, (width,), params[1], params[2])
    want = torch.nn.functional.cross_entropy((h @ params[0].t()).flatten(0, 1), targets.flatten(), ignore_index=ex.PAD)
    want.backward()
    want = want.detach()
    assert abs(float(loss) - float(want)) <= 2.0**-6 * float(want)
    for got, p in zip(grads, params):
        assert got.dtype == torch.float32
        assert float((got.double() - p.grad).norm()) <= 2.0**-4 * float(p.grad.norm())


def test_learns():
    """From about log(vocabulary) to below half of it (0.1 log(vocabulary) +
    0.33 is the text's own entropy)."""
    ex = _example()
    vocab = 512
    first, held = ex.train(steps=60, tokens=4096, vocab=vocab, width=128, report=0)
    assert 0.5 * math.log(vocab) < first
    assert held < 0.5 * math.log(vocab)
