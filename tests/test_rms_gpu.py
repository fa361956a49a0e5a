"""The root-mean-square norm of hc.gfx950 and its gradient on the GPU against
plain definitions in 64 bits.

Tolerances are forward error bounds.  A float32 sum here runs over a lane's
values, then lanes, then waves: DEPTH(width) additions deep, each within 2^-24
of its result, so a sum of squares is within that many 2^-24 of itself, and
rstd within half as many, two more for the division and the root, and one for
the product with eps' sum.  u is a type's unit roundoff."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc._errors import LaunchError  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0**-11, BF16: 2.0**-8, F32: 2.0**-24}
TINY = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}  # half the smallest step near zero
E32 = 2.0**-24
TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (BF16, F32), (F16, F32)]
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (33, 127), (7, 128), (9, 129), (300, 256), (31, 515), (64, 1024),
          (70, 1027), (17, 2048), (6, 4100), (1000, 72), (3, 8192), (5, 16384), (2, 32768), (2, 40001)]


def _depth(width):
    return 40 + width // 256


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std + mean).to(dtype)


def _strided(t, pad, offset=0):
    """t's values as a view with rows `pad` elements longer, NaN around it."""
    rows, width = t.shape
    buf = torch.full((rows * (width + pad) + offset + 8,), float("nan"), dtype=t.dtype, device=t.device)
    view = buf[offset : offset + rows * (width + pad)].view(rows, width + pad)[:, :width]
    view.copy_(t)
    return view


def _close(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (
        f"{int(bad.sum())} of {got.numel()} outside the bound; worst {float((got - want).abs().max()):.3g}, "
        f"first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])}")


@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, width, dtype, wide, residual):
    gen = _gen(rows * 31 + width)
    x = _strided(_randn(gen, (rows, width), dtype), 3, 1)
    res = _strided(_randn(gen, (rows, width), wide, 2.0, 0.5), 5, 2) if residual else None
    weight = _randn(gen, (width,), wide, 0.1, 1.0)
    y, h, rstd = g.rms_norm(x, weight, res, eps=1e-5)
    assert y.dtype == dtype and rstd.dtype == F32 and y.shape == x.shape and rstd.shape == (rows,)
    if residual:
        assert h.dtype == wide and torch.equal(h, (x.float() + res.float()).to(wide))
    else:
        assert h is x
    hd = h.double()
    want = (hd.square().mean(1) + 1e-5).rsqrt()
    rel = (_depth(width) / 2 + 4) * E32
    _close(rstd, want, rel * want)
    ywant = hd * want[:, None] * weight.double()
    _close(y, ywant, (rel + 2 * E32 + U[dtype]) * ywant.abs() + TINY[dtype])


@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(600, 1536), (520, 2560), (3000, 40), (1025, 4096)])
def test_grad(rows, width, dtype, wide):
    gen = _gen(rows * 17 + width)
    dy = _strided(_randn(gen, (rows, width), dtype), 3, 1)
    h = _strided(_randn(gen, (rows, width), wide, 2.0, 0.5), 5, 2)
    dres = _strided(_randn(gen, (rows, width), wide, 3.0), 1, 3)
    weight = _randn(gen, (width,), dtype, 0.1, 1.0)
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    dh, dweight = g.rms_norm_grad(dy, h, rstd, weight, dresidual=dres)
    assert dh.dtype == wide and dweight.dtype == dtype
    d, x, r, w = dy.double(), h.double(), rstd.double()[:, None], weight.double()
    xh, gw = x * r, dy.double() * w
    dot = (gw * xh).mean(1, keepdim=True)
    mag = (gw * xh).abs().mean(1, keepdim=True)  # the dot's rounding, by the sum of magnitudes
    want = r * (gw - xh * dot) + dres.double()
    inner = r * (gw.abs() + xh.abs() * mag)
    _close(dh, want, ((_depth(width) + 8) * E32) * inner + 2 * E32 * want.abs() + U[wide] * want.abs() + TINY[wide])
    # columns: up to rows / 256 turns, then at most 32 groups, 16 + 16 parts
    dwant, dmag = (d * xh).sum(0), (d * xh).abs().sum(0)
    _close(dweight, dwant, (rows / 64 + 80) * E32 * dmag + U[dtype] * dwant.abs() + TINY[dtype])
    # float32 sums on demand, of the same weight
    wide_dh, wide_dw = g.rms_norm_grad(dy, h, rstd, weight, dresidual=dres, param_dtype=F32)
    assert torch.equal(wide_dh, dh) and wide_dw.dtype == F32 and torch.equal(wide_dw.to(dtype), dweight)
    # nothing past the norm, no weight
    plain, _ = g.rms_norm_grad(dy, h, rstd)
    pdot, pmag = (d * xh).mean(1, keepdim=True), (d * xh).abs().mean(1, keepdim=True)
    pwant = r * (d - xh * pdot)
    _close(plain, pwant, ((_depth(width) + 8) * E32) * r * (d.abs() + xh.abs() * pmag) + U[wide] * pwant.abs() + TINY[wide])


# Rows that end inside a vector, several to a row group.
@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("rows,width", [(4000, 5), (9000, 13), (5000, 130), (2601, 517), (2001, 1027), (521, 4101), (258, 8197)])
def test_grad_ragged_turns(rows, width, dtype, wide):
    test_grad(rows, width, dtype, wide)


def test_grad_against_differences():
    """The gradient of sum(c * norm(x)) along a direction, by central
    differences of the forward call in float32."""
    gen = _gen(5)
    rows, width = 6, 96
    x, res, c, v = (_randn(gen, (rows, width), F32) for _ in range(4))
    weight, dw_dir = _randn(gen, (width,), F32, 0.1, 1.0), _randn(gen, (width,), F32)
    _, h, rstd = g.rms_norm(x, weight, res)
    dh, dweight = g.rms_norm_grad(c, h, rstd, weight)

    def value(step):
        y, _, _ = g.rms_norm(x + step * v, weight + step * dw_dir, res)
        return float((y.double() * c.double()).sum())

    step = 2.0**-7
    slope = (value(step) - value(-step)) / (2 * step)
    want = float((dh.double() * v.double()).sum() + (dweight.double() * dw_dir.double()).sum())
    # third derivatives of order 1 per element times step^2 / 6, and float32's rounding over the step
    scale = float((c.abs() * (v.abs() + 1) ** 3).sum())
    assert abs(slope - want) <= scale * (step * step + 16 * E32 / step)


def test_special_rows():
    """Rows of zeros, infinities and NaNs, and rows beside them."""
    x = torch.zeros((5, 300), dtype=BF16, device=DEV)
    x[1] = 1.0
    x[2, 7] = float("inf")
    x[3, 299] = float("nan")
    x[4] = -2.0
    y, h, rstd = g.rms_norm(x, eps=1e-6)
    assert (y[0] == 0).all() and abs(float(rstd[0]) - 1000) < 1e-3
    assert (y[1] == 1).all() and (y[4] == -1).all()
    assert y[2, 7].isnan() and (y[2, :7] == 0).all() and float(rstd[2]) == 0
    assert y[3].isnan().all()


def test_shapes_and_empty():
    gen = _gen(1)
    x = _randn(gen, (2, 3, 40), BF16)
    res = _randn(gen, (2, 3, 40), F32)
    y, h, rstd = g.rms_norm(x, None, res)
    assert y.shape == h.shape == (2, 3, 40) and rstd.shape == (2, 3)
    flat, fh, frstd = g.rms_norm(x.view(6, 40), None, res.view(6, 40))
    assert torch.equal(y.view(6, 40), flat) and torch.equal(h.view(6, 40), fh) and torch.equal(rstd.view(6), frstd)
    one, _, r = g.rms_norm(x[0, 0])
    assert one.shape == (40,) and r.shape == ()
    for t in (x.transpose(0, 1), x[:, ::2], x[..., ::2]):
        a, _, _ = g.rms_norm(t)
        b, _, _ = g.rms_norm(t.contiguous())
        assert torch.equal(a, b)
    empty, eh, er = g.rms_norm(x[:, :0], None, res[:, :0])
    assert empty.shape == eh.shape == (2, 0, 40) and er.shape == (2, 0)
    dh, dw = g.rms_norm_grad(x[:, :0], res[:, :0], er)
    assert dh.shape == (2, 0, 40) and dw.shape == (40,) and (dw == 0).all()


def test_out():
    gen = _gen(2)
    x = _randn(gen, (9, 50), F16)
    want, _, _ = g.rms_norm(x)
    buf = torch.full((9, 60), 7.0, dtype=F16, device=DEV)
    got, _, _ = g.rms_norm(x, out=buf[:, 4:54])
    assert got.data_ptr() == buf[:, 4:].data_ptr() and torch.equal(got, want)
    assert (buf[:, :4] == 7).all() and (buf[:, 54:] == 7).all()
    turned = torch.empty((50, 9), dtype=F16, device=DEV)
    assert torch.equal(g.rms_norm(x, out=turned.t())[0], want) and torch.equal(turned.t(), want)


@pytest.mark.parametrize("call,match", [
    (lambda x, r: g.rms_norm(x, r[0, :9]), "width"), (lambda x, r: g.rms_norm(x, r[0].double()), "weight must be"),
    (lambda x, r: g.rms_norm(x, None, r[:3]), "residual shape"), (lambda x, r: g.rms_norm(x, None, r.half()), "residual must"),
    (lambda x, r: g.rms_norm(x.double()), "x must be"), (lambda x, r: g.rms_norm(x[:, :0]), "without elements"),
    (lambda x, r: g.rms_norm(x, out=r), "out must be"), (lambda x, r: g.rms_norm(x, None, r.cpu()), "GPU"),
    (lambda x, r: g.rms_norm_grad(x, r[:3], r[:, 0]), "does not match h"),
    (lambda x, r: g.rms_norm_grad(x, r, r[:3, 0]), "rstd must"),
    (lambda x, r: g.rms_norm_grad(x, r, r[:, 0], dresidual=x), "dresidual must"),
    (lambda x, r: g.rms_norm_grad(x, x.half(), r[:, 0]), "h must be"),
    (lambda x, r: g.rms_norm_grad(x, r, r[:, 0], param_dtype=F16), "param_dtype")])
def test_refusals(call, match):
    x = torch.ones((4, 16), dtype=BF16, device=DEV)
    with pytest.raises(LaunchError, match=match):
        call(x, torch.ones((4, 16), device=DEV))


def test_graph_and_streams():
    """Captured once and replayed over new inputs, on a stream of its own."""
    gen = _gen(3)
    x, res, dy = (_randn(gen, (40, 512), BF16) for _ in range(3))
    weight = _randn(gen, (512,), BF16, 0.1, 1.0)

    def call():
        y, h, rstd = g.rms_norm(x, weight, res)
        return (y, h, rstd, *g.rms_norm_grad(dy, h, rstd, weight, dresidual=res))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for i in range(3):
        x.copy_(_randn(gen, (40, 512), BF16))
        dy.copy_(_randn(gen, (40, 512), BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            want = call()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
