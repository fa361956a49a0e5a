"""hc.gfx950.linear_cross_entropy and its gradient: probabilities far below
the largest, and sizes that reach every tile shape of the three products (on
the host test_lm_plan.py asks the library that they do)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc._errors import LaunchError  # noqa: E402

from .test_lm_gpu import (BF16, DEV, E32, F16, F32, TINY, U, _close, _gen, _grad_tols, _head, _head_want,  # noqa: E402
                          _loss_tol, _twice)

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


# Tokens, vocabulary, width: with those of test_lm_gpu.py every tile shape of
# logits, dx and dweight, with and without split sums; ragged on all sides, and
# in whole tiles; the last one in two pieces of large tiles.
HEADS = [(432, 31059, 200), (2707, 413, 3416), (3861, 27862, 133), (3000, 3000, 3000), (1999, 50021, 1027),
         (2048, 32768, 1024), (3138, 20, 1922), (36, 5794, 4089), (618, 16, 19), (3450, 17, 1159), (68, 39280, 19),
         (4500, 131072, 264)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t,v,d", HEADS)
def test_loss_by_every_tile_shape(t, v, d, dtype):
    x, w, y = _head(t, v, d, dtype, t + v + d)
    keep = torch.rand((t,), generator=_gen(t), device=DEV) < 0.9
    x[~keep] = float("nan")  # ignored rows may hold anything
    lse, loss, slack, _, _ = _head_want(x, w, y, keep)
    got = _twice(lambda: g.linear_cross_entropy(x, w, torch.where(keep, y, -100)))
    tol = _loss_tol(slack, lse)
    for a, b in zip(got, (loss, lse)):
        assert a.shape == (t,) and a.dtype == F32 and (a[~keep] == 0).all()
        _close(a[keep], b[keep], tol[keep])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("share", [0.8, 0.1])  # (few that count: the device splits sums into more parts than the host planned)
@pytest.mark.parametrize("t,v,d", HEADS)
def test_gradient_by_every_tile_shape(t, v, d, share, dtype):
    x, w, y = _head(t, v, d, dtype, 2 * t + v + d)
    keep = torch.rand((t,), generator=_gen(t), device=DEV) < share
    x[~keep] = float("nan")
    lse, loss, slack, gz, p = _head_want(x, w, y, keep)
    got = _twice(lambda: g.linear_cross_entropy_grad(x, w, torch.where(keep, y, -100), reduction="sum"))
    assert got[0].shape == () and got[1].dtype == got[2].dtype == dtype
    tol = _loss_tol(slack, lse)[keep].sum() + (t / 1024 + 30) * E32 * loss[keep].abs().sum()
    assert abs(float(got[0]) - float(loss[keep].sum())) <= float(tol)
    (dx, tx), (dw, tw) = _grad_tols(x, w, gz, p, slack, keep, 1.0, dtype)
    _close(got[1], dx, tx)
    _close(got[2], dw, tw)
    assert (got[1][~keep] == 0).all()


def test_refuses_an_ignored_target_that_no_target_can_be():
    x, w, y = _head(4, 9, 8, BF16, 0)
    for bad in (1.5, "-100", None, 2**63, 2**64 - 100):
        for call in (g.linear_cross_entropy, g.linear_cross_entropy_grad):
            with pytest.raises(LaunchError, match="ignore_index must be a whole number"):
                call(x, w, y, ignore_index=bad)
