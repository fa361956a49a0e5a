"""hc.gfx950.layer_norm and its gradient: parameters of other types than the
rows, and rows whose padding could reach a sum."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

from .test_lm_gpu import BF16, DEV, E32, F16, F32, TINY, U, _close, _gen, _K, _randn  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,width", [(3, 40), (50, 1027), (2, 16400)])
def test_param_dtype_is_the_gradients_type_only(rows, width, dtype):
    """A float32 weight that no 16-bit type holds (and one past float16's
    range) enters dx as it is; only dweight and dbias are rounded."""
    gen = _gen(rows + width)
    x, dy = _randn(gen, (rows, width), dtype), _randn(gen, (rows, width), dtype, 2.0**-6)
    w = 1 + torch.rand((width,), generator=gen, device=DEV) * 2.0**-10
    w[width // 2] = 70001.0
    _, mean, rstd = g.layer_norm(x, w)
    dx, dw, db = g.layer_norm_grad(dy, x, mean, rstd, w)
    assert dw.dtype == db.dtype == F32 and dx.isfinite().all()
    got = g.layer_norm_grad(dy, x, mean, rstd, w, param_dtype=dtype)
    assert got[1].dtype == got[2].dtype == dtype and got[1].shape == got[2].shape == (width,)
    for a, b in zip(got, (dx, dw.to(dtype), db.to(dtype))):
        assert torch.equal(a, b)
    # without rows: zeros of the type asked for
    e, s = x[:0], mean[:0]
    got = g.layer_norm_grad(e, e, s, s, w, param_dtype=dtype)
    assert got[1].dtype == got[2].dtype == dtype and (got[1] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("dtype,width,value,eps", [(F32, 5, 2.0**123, 1e-5), (BF16, 13, 2.0**122, 1e-5),
                                                   (F32, 1027, 2.0**100, 1e-24), (BF16, 2500, 2.0**100, 1e-24),
                                                   (F32, 8195, 2.0**100, 1e-24), (BF16, 16397, 2.0**100, 1e-24)])
def test_gradient_of_large_equal_values(dtype, width, value, eps):
    """Rows of one value so large that -mean * rstd overflows: xhat is 0 in
    every column, and what lies past the last column reaches no sum."""
    gen = _gen(width)
    x = torch.full((3, width), value, dtype=dtype, device=DEV)
    dy = _randn(gen, (3, width), dtype)
    w = _randn(gen, (width,), F32, 0.2, 1.0)
    _, mean, rstd = g.layer_norm(x, w, eps=eps)
    assert (mean == value).all() and (mean * rstd).isinf().all()
    dx, dw, db = g.layer_norm_grad(dy, x, mean, rstd, w)
    gw, rs = dy.double() * w.double(), rstd.double()[:, None]
    want = rs * (gw - gw.mean(1, keepdim=True))
    tol = _K * E32 * rs * 2 * gw.abs().amax(1, keepdim=True)
    _close(dx, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    assert (dw == 0).all()
    _close(db, dy.double().sum(0), 5 * E32 * dy.double().abs().sum(0))
