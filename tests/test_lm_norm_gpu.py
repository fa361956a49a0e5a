"""hc.gfx950.layer_norm and its gradient: parameters of other types than the
rows."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

from .test_lm_gpu import BF16, DEV, F16, F32, _gen, _randn  # noqa: E402

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
