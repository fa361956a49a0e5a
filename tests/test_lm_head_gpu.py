"""hc.gfx950.linear_cross_entropy and its gradient: probabilities far below
the largest."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

from .test_lm_gpu import BF16, DEV, E32, F16, TINY, U, _close, _head_want  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t,v,base", [(1, 60, 0.0), (1, 60, -40.0), (200, 300, 0.0), (40, 5000, 3.0), (130, 300, 2.0**21)])
def test_small_probabilities_keep_their_gradient(t, v, base, dtype):
    """Logits from `base` down in steps of a half, in runs of 60 words:
    probabilities to 2^-42 of the largest.  A probability carries its
    exponentials' errors (2^-18), their 16-bit form (2^-11, or 2^-40 of the
    block's largest) and the rounding to the operands' type (float16: times
    2^15, so 2^-40 near zero).  Past exponents of 2^20 the 16-bit form is held to 2^-25 of the largest."""
    d = 16
    x = torch.zeros((t, d), dtype=dtype, device=DEV)
    x[:, 0], x[:, 1] = 1.0, 2.0**7
    w = torch.zeros((v, d), dtype=dtype, device=DEV)
    w[:, 0] = -(torch.arange(v, device=DEV) % 60).to(dtype) / 2
    w[:, 1] = base / 2**7
    y = torch.zeros((t,), dtype=torch.int64, device=DEV)
    keep = torch.ones((t,), dtype=torch.bool, device=DEV)
    _, _, _, gz, p = _head_want(x, w, y, keep)
    scale = 2.0**16 / t
    _, _, dw = g.linear_cross_entropy_grad(x, w, y, reduction="sum", grad_scale=scale)
    rel = 2.0**-18 + 2.0**-11 + t * E32
    eps = rel * p + U[dtype] * gz.abs() * (1 + rel) + (2.0**-39 if base < 2**20 else 2.0**-24)
    want, tol = gz.sum(0) * scale, eps.sum(0) * scale
    _close(dw[:, 0], want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
