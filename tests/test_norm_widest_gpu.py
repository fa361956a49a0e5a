"""Rows so wide that a launch's threads along one dimension do not number their
columns' sums: the gradients of both norms.

dy and h (or x) are whole numbers of -1 to 1 and the statistics 1 and 0, so that a
column's sum of one row is exact, and so is the row's dot product (a sum of less
than 2^24 in whole numbers).  What is left is one float32 division by the width,
one product, one subtraction and the result's own rounding."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
STEP = 1 << 26  # columns compared at a time


def _signs(gen, width):
    t = torch.empty((1, width), dtype=F16, device=DEV)
    for at in range(0, width, STEP):
        part = t[:, at : at + STEP]
        part.copy_(torch.randint(-1, 2, part.shape, generator=gen, device=DEV, dtype=torch.int8))
    return t


def _dot(a, b, width):
    return sum(float((a[:, at : at + STEP].float() * b[:, at : at + STEP].float()).sum(dtype=torch.float64))
               for at in range(0, width, STEP))


@pytest.mark.parametrize("width", [(1 << 28) - 64, (1 << 28) + 5, 1 << 30])
def test_rms_norm_grad(width):
    gen = torch.Generator(device=DEV).manual_seed(1)
    dy, h = _signs(gen, width), _signs(gen, width)
    dh, dweight = g.rms_norm_grad(dy, h, torch.ones((1,), device=DEV))
    mean = _dot(dy, h, width) / width
    assert abs(mean) < 2.0**-5
    for at in range(0, width, STEP):
        d, x = dy[:, at : at + STEP].double(), h[:, at : at + STEP].double()
        assert torch.equal(dweight[at : at + STEP].double(), (d * x)[0])
        # |d - x mean| < 2, so half a step of float16 is at most 2^-11, and float32's three roundings 3 * 2^-24
        assert float((dh[:, at : at + STEP].double() - (d - x * mean)).abs().max()) <= 2.0**-11 + 3 * 2.0**-24


@pytest.mark.parametrize("width", [(1 << 28) - 64, (1 << 28) + 5])
def test_layer_norm_grad(width):
    gen = torch.Generator(device=DEV).manual_seed(2)
    dy, x = _signs(gen, width), _signs(gen, width)
    one = torch.ones((1,), device=DEV)
    dx, dweight, dbias = g.layer_norm_grad(dy, x, torch.zeros_like(one), one)
    along = _dot(dy, x, width) / width
    mean = sum(float(dy[:, at : at + STEP].sum(dtype=torch.float64)) for at in range(0, width, STEP)) / width
    assert abs(mean) + abs(along) < 2.0**-5
    assert torch.equal(dbias, dy[0])
    for at in range(0, width, STEP):
        d, v = dy[:, at : at + STEP].double(), x[:, at : at + STEP].double()
        assert torch.equal(dweight[at : at + STEP].double(), (d * v)[0])
        # as above, with a division and a subtraction more
        assert float((dx[:, at : at + STEP].double() - (d - mean - v * along)).abs().max()) <= 2.0**-11 + 5 * 2.0**-24
