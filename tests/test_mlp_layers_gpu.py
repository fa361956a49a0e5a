"""The example of 8-bit linear layers with two blocks: the gradients that pass
from block to block, against autograd in 64 bits."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests.test_mlp_example_gpu import _example  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,width,rows,length", [(300, 72, 9, 31), (500, 128, 3, 50)])
def test_gradients_of_two_blocks(vocab, width, rows, length):
    """By norms.  A quantised operand errs by at most u / sqrt(3) of its norm, u =
    2^-4 (e4m3) or 2^-3 (e5m2): 0.036 and 0.072.  A block's result has a product
    whose square is taken (2 * 0.036 * sqrt(2) = 0.102), its own quantisation and
    the second weight's: 0.114.  A gradient passes three products of a block
    (0.081 each: an operand of either type) and the square's factor (0.051).  Both
    blocks' errors enter the first one's gradients, independently: sqrt(2 * (0.114^2
    + 3 * 0.081^2 + 0.051^2)) = 0.27; the bound is twice that, for parameters of few
    values.  A path from block to block left out, or of the wrong sign, is an error
    of the gradient's own size."""
    ex = _example()
    gen = torch.Generator(device="cuda:0").manual_seed(4)
    model = ex.Model(vocab, width, 2, "cuda:0")
    tokens, targets = ex.text(rows, length, torch.randperm(vocab, generator=gen, device="cuda:0"), gen)
    loss, grads = model.loss_and_grads(tokens, targets)
    p = [q.double().requires_grad_() for q in model.params]

    def norm(h, w):
        return h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    h = p[0][tokens] * model.scale
    for i in (1, 4):
        h = h + (norm(h, p[i]) @ p[i + 1].t()).relu().square() @ p[i + 2].t()
    want = torch.nn.functional.cross_entropy((norm(h, p[7]) @ p[0].t()).flatten(0, 1), targets.flatten(),
                                             ignore_index=ex.PAD)
    want.backward()
    assert len(grads) == len(p) == 8
    for got, q in zip(grads, p):
        assert got.dtype == torch.float32 and got.shape == q.shape
        assert float((got.double() - q.grad).norm()) <= 0.54 * float(q.grad.norm())
