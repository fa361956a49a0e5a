"""The root-mean-square norm's C entry points where Python's never go: the sum
written over the residual, the gradient over the one that reaches it past the
norm, and calls without what may be left out.  Every result is that of a call with
everything in memory of its own, bit for bit."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc.gfx950 import _native  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
CODES = {F16: _native.HCG_F16, BF16: _native.HCG_BF16, F32: _native.HCG_F32}
TYPES = [(F16, F16), (BF16, F32), (F32, F32)]
# Rows in registers of a part of a wave, a wave, several; rows that end inside a
# vector; several turns of the gradient's loop; wide ones.
SHAPES = [(1, 1), (7, 3), (2000, 5), (33, 64), (5000, 130), (1200, 517), (9, 1027), (1025, 4096), (300, 8197), (270, 16383),
          (5, 40001)]


def _inputs(rows, width, dtype, wide):
    gen = torch.Generator(device=DEV).manual_seed(rows + width)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    return (randn(rows, width).to(dtype), (randn(rows, width) * 2).to(wide), randn(rows, width).to(wide),
            (randn(width) * 0.1 + 1).to(dtype))


def _framed(t, pad):
    """t's values in rows `pad` elements longer, 7 in between, and the whole."""
    buf = torch.full((t.shape[0], t.shape[1] + pad), 7.0, dtype=t.dtype, device=DEV)
    buf[:, : t.shape[1]] = t
    return buf[:, : t.shape[1]], buf


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("pad", [0, 3])
def test_sum_over_the_residual(rows, width, dtype, wide, pad):
    x, res, _, weight = _inputs(rows, width, dtype, wide)
    want_y, want_h, want_rstd = g.rms_norm(x, weight, res)
    want_q, want_s, _, _ = g.rms_norm_fp8(x, weight, res)
    lib = _native.lib()
    for rstd in (torch.empty((rows,), device=DEV), None):
        at = rstd.data_ptr() if rstd is not None else None
        held, buf = _framed(res, pad)
        y = torch.empty_like(x)
        rc = lib.hcg_rms_norm(CODES[dtype], x.data_ptr(), width, rows, width, CODES[wide], held.data_ptr(), width + pad,
                              CODES[dtype], weight.data_ptr(), 1e-6, y.data_ptr(), width, held.data_ptr(), width + pad, at,
                              _stream())
        assert rc == 0 and torch.equal(y, want_y) and torch.equal(held, want_h) and (buf[:, width:] == 7).all()
        assert rstd is None or torch.equal(rstd, want_rstd)
        held, buf = _framed(res, pad)
        q, s = torch.empty((rows, width), dtype=want_q.dtype, device=DEV), torch.empty(want_s.shape, device=DEV)
        rc = lib.hcg_rms_norm_fp8(CODES[dtype], x.data_ptr(), width, rows, width, CODES[wide], held.data_ptr(), width + pad,
                                  CODES[dtype], weight.data_ptr(), 1e-6, _native.HCG_E4M3, q.data_ptr(), width,
                                  _native.HCG_F32, s.data_ptr(), s.stride(0), 1, held.data_ptr(), width + pad, at, _stream())
        assert rc == 0 and torch.equal(held, want_h) and (buf[:, width:] == 7).all() and torch.equal(s, want_s)
        assert torch.equal(q.view(torch.uint8), want_q.contiguous().view(torch.uint8))
        assert rstd is None or torch.equal(rstd, want_rstd)


@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("pad", [0, 3])
def test_gradient_over_the_one_past_the_norm(rows, width, dtype, wide, pad):
    dy, h, dres, weight = _inputs(rows, width, dtype, wide)
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    want, want_dw = g.rms_norm_grad(dy, h, rstd, weight, dresidual=dres)
    lib = _native.lib()
    need = lib.hcg_rms_norm_grad_workspace(rows, width)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    for dw in (torch.empty_like(want_dw), None):  # (without it no scratch either)
        held, buf = _framed(dres, pad)
        rc = lib.hcg_rms_norm_grad(CODES[dtype], dy.data_ptr(), width, CODES[wide], h.data_ptr(), width, rows, width,
                                   rstd.data_ptr(), CODES[dtype], weight.data_ptr(), held.data_ptr(), width + pad,
                                   held.data_ptr(), width + pad, None if dw is None else dw.data_ptr(),
                                   None if dw is None else ws.data_ptr(), 0 if dw is None else need, _stream())
        assert rc == 0 and torch.equal(held, want) and (buf[:, width:] == 7).all()
        assert dw is None or torch.equal(dw, want_dw)
