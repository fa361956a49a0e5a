"""hc.gfx950.layer_norm and its gradient: parameters of other types than the
rows, rows whose padding could reach a sum, and row counts at which every form
of the gradient's kernel takes several turns."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

from .test_lm_gpu import BF16, DEV, E32, F16, F32, TINY, U, _close, _gen, _K, _norm_want, _randn, _twice  # noqa: E402

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


# (width in vectors of 16 bytes, rows of a turn of 256 workgroups): every form
# of the gradient's kernel, with widths that end inside a vector.
_FORMS = [(15, 8192), (31, 4096), (60, 2048), (127, 2048), (191, 1280), (255, 1024), (319, 768), (361, 512),
          (511, 512), (1000, 256), (2047, 256)]


def _grad_check(rows, width, dtype, pdtype):
    gen = _gen(rows * 5 + width)
    x, dy = _randn(gen, (rows, width), dtype, 1.5, 0.5), _randn(gen, (rows, width), dtype)
    w = _randn(gen, (width,), pdtype, 0.2, 1.0)
    _, m, r, _ = _norm_want(x, w, None, 1e-5)
    mean, rstd = m[:, 0].float(), r[:, 0].float()
    dx, dw, db = _twice(lambda: g.layer_norm_grad(dy, x, mean, rstd, w))
    assert dx.dtype == dtype and dw.dtype == db.dtype == pdtype
    rs = rstd.double()[:, None]
    xh = (x.double() - mean.double()[:, None]) * rs
    gw = dy.double() * w.double()
    want = rs * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    top, far = gw.abs().amax(1, keepdim=True), xh.abs().amax(1, keepdim=True)
    # xh from float32 mean and rstd: 3 roundings of (|x| + |mean|) rstd
    far = far + 4 * E32 * rs * (x.double().abs().amax(1, keepdim=True) + mean.double().abs()[:, None])
    tol = _K * E32 * rs * top * (2 + far + far * far)
    _close(dx, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    del want, gw
    # A column's chain: a row per turn, the groups (at most 32), the parts.
    chain = rows / 128 + 300
    big = rs * (x.double().abs() + mean.double().abs()[:, None])
    for got, wt, mag in ((dw, (dy.double() * xh).sum(0), (dy.double().abs() * (xh.abs() + big)).sum(0)),
                         (db, dy.double().sum(0), dy.double().abs().sum(0))):
        tol = chain * E32 * mag
        _close(got, wt, tol + U[pdtype] * (wt.abs() + tol) + TINY[pdtype])


@pytest.mark.parametrize("dtype,pdtype", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("turns", [1, 2, 3, 5])
@pytest.mark.parametrize("vecs,per_turn", _FORMS)
def test_gradient_over_several_turns(vecs, per_turn, turns, dtype, pdtype):
    """`turns` turns, the last of a third of the rows; 1: one turn and a row."""
    elems = 4 if dtype == F32 else 8
    _grad_check(per_turn * (turns - 1) + (per_turn // 3 if turns > 1 else per_turn) + 1, vecs * elems - 3, dtype, pdtype)


@pytest.mark.parametrize("rows,width,dtype", [
    (512, 4096, BF16), (511, 4096, F16), (1024, 4096, BF16),       # whole turns, and a row short of one
    (4100, 4096, BF16), (4104, 2048, F32), (70000, 320, F16),      # dx past 32 MB in whole 128-byte lines
    (130, 16400, BF16), (65, 8196, F32), (200, 16385, F16)])       # past registers: columns over several rows
def test_gradient_of_many_rows(rows, width, dtype):
    _grad_check(rows, width, dtype, dtype)


@pytest.mark.parametrize("rows,width", [(40000, 128), (5000, 1027), (300, 16400)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forward_of_many_rows(rows, width, dtype):
    gen = _gen(rows)
    x = _randn(gen, (rows, width), dtype, 1.5, 0.5)
    w, b = _randn(gen, (width,), F32, 0.2, 1.0), _randn(gen, (width,), F32, 0.3)
    y, mean, rstd = _twice(lambda: g.layer_norm(x, w, b))
    wy, wm, wr, _ = _norm_want(x, w, b, 1e-5)
    top = x.double().abs().amax(1, keepdim=True)
    _close(mean[:, None], wm, _K * E32 * top)
    _close(rstd[:, None], wr, _K * E32 * (wr + wr**3 * top * top))
    tol = _K * E32 * ((wr + wr**3 * top * top) * 2 * top * w.double().abs() + b.double().abs())
    _close(y, wy, tol + U[dtype] * (wy.abs() + tol) + TINY[dtype])
