"""The language-model operators of hc.gfx950 on the GPU against plain
definitions in 64 bits.

Tolerances are forward error bounds: u is a type's unit roundoff (half the
spacing at 1), float32 sums of k terms are within k * 2^-24 of the sum of
magnitudes, and each intermediate that is held in fewer bits adds its own
rounding.  Results held to no bound are compared bit for bit."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc._errors import LaunchError  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0**-11, BF16: 2.0**-8, F32: 2.0**-24}
TINY = {F16: 2.0**-25, BF16: 0.0, F32: 0.0}  # half the smallest step near zero
E32 = 2.0**-24


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


def _twice(call):
    """The call's results, which are the same bits the second time."""
    a, b = call(), call()
    for x, y in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
        assert torch.equal(x.view(torch.uint8) if x.ndim else x, y.view(torch.uint8) if y.ndim else y)
    return a


# --------------------------------------------------------------------------
# Embedding
# --------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 5, 64), (7, 100, 515), (1000, 37, 8), (3, 11, 40001),
                                           (300, 257, 1024)])
def test_embedding(n, vocab, width, ids, dtype):
    gen = _gen(n + vocab + width)
    table = _strided(_randn(gen, (vocab, width), dtype), 3, 1)
    tokens = torch.randint(0, vocab, (n,), generator=gen, device=DEV).to(ids)
    scale = 1.7
    out = g.embedding(tokens, table, scale=scale)
    assert torch.equal(out, (table[tokens.long()].float() * scale).to(dtype))
    # into a strided view: nothing around it changes
    buf = torch.full((n, width + 5), 7.0, dtype=dtype, device=DEV)
    assert g.embedding(tokens, table, scale=scale, out=buf[:, 2 : 2 + width]).data_ptr() == buf[:, 2:].data_ptr()
    assert torch.equal(buf[:, 2 : 2 + width], out)
    assert (buf[:, :2] == 7).all() and (buf[:, 2 + width :] == 7).all()


def test_embedding_shapes_and_unknown_tokens():
    table = _randn(_gen(0), (10, 16), BF16)
    tokens = torch.tensor([[3, -1, 9], [10, 0, 1 << 40]], device=DEV)
    out = g.embedding(tokens, table)
    assert out.shape == (2, 3, 16)
    known = torch.tensor([[True, False, True], [False, True, False]], device=DEV)
    assert torch.equal(out[known], table[tokens[known]])
    assert out[~known].isnan().all()
    assert g.embedding(tokens[:, :0], table).shape == (2, 0, 16)
    assert torch.equal(g.embedding(tokens[0, ::2], table), table[tokens[0, ::2]])
    assert torch.equal(g.embedding(torch.tensor(4, device=DEV), table), table[4])
    assert torch.equal(g.embedding(tokens[0, ::2], table[::2, ::3]), torch.stack([table[6, ::3], table[9, ::3] * float("nan")]))\
        or g.embedding(tokens[0, ::2], table[::2, ::3])[1].isnan().all()


def _embedding_grad_want(dy, tokens, vocab, scale, padding=None):
    keep = (tokens >= 0) & (tokens < vocab)
    if padding is not None:
        keep &= tokens != padding
    t, d = tokens[keep].long(), dy[keep].double()
    want = torch.zeros((vocab, dy.shape[1]), dtype=torch.float64, device=DEV).index_add_(0, t, d) * scale
    mag = torch.zeros_like(want).index_add_(0, t, d.abs()) * abs(scale)
    count = torch.zeros((vocab,), dtype=torch.float64, device=DEV).index_add_(0, t, torch.ones_like(t, dtype=torch.float64))
    return want, mag, count[:, None]


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (BF16, BF16), (F32, F32), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("n,vocab,width,spread", [
    (1, 1, 1, "even"), (0, 7, 12, "even"), (1, 300, 70, "even"), (32, 1, 16, "even"), (33, 1, 16, "even"),
    (64, 3, 515, "even"), (65, 1, 9, "even"), (97, 1, 4100, "even"), (1000, 37, 40, "zipf"), (999, 5003, 515, "zipf"),
    (5000, 70001, 24, "zipf"), (3000, 900, 64, "one"), (2100, 3, 130, "even"), (4099, 129, 33, "edges")])
def test_embedding_grad(n, vocab, width, spread, dtype, out_dtype):
    gen = _gen(n * 7 + vocab + width)
    u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
    if spread == "even":
        tokens = (u * vocab).long().clamp_(max=vocab - 1)
    elif spread == "one":  # nearly all the same row
        tokens = torch.where(u < 0.97, vocab // 2, (u * 31337).long() % vocab)
    elif spread == "edges":  # runs that end on, before and after a window's edge, and unknown ids on both sides
        lengths = [31, 32, 33, 34, 63, 64, 65, 66, 127, 128, 129, 1, 200]
        ids = [i for i, c in enumerate(lengths) for _ in range(c)]
        tokens = torch.full((n,), -5, device=DEV)
        tokens[: len(ids)] = torch.tensor(ids, device=DEV) * 9
        tokens[len(ids) : len(ids) + 100] = vocab + 3
        tokens = tokens[torch.randperm(n, generator=gen, device=DEV)]
    else:
        tokens = ((torch.exp(u * math.log(vocab + 1.0)) - 1).long() * 7919 % vocab).clamp_(0, vocab - 1)
    dy = _strided(_randn(gen, (n, width), dtype), 5, 1) if n else torch.empty((0, width), dtype=dtype, device=DEV)
    scale = 1.5
    got = _twice(lambda: g.embedding_grad(dy, tokens, vocab, scale=scale, dtype=out_dtype))
    assert got.dtype == out_dtype and got.shape == (vocab, width)
    want, mag, count = _embedding_grad_want(dy, tokens, vocab, scale)
    _close(got, want, (count + 2) * E32 * mag + U[out_dtype] * want.abs() + TINY[out_dtype])
    assert (got[(count[:, 0] == 0)] == 0).all()


def test_embedding_grad_padding_row_and_view():
    gen = _gen(5)
    tokens = torch.randint(0, 40, (4, 100), generator=gen, device=DEV, dtype=torch.int32)
    dy = _randn(gen, (4, 100, 48), F32)
    dy[tokens == 6] = float("nan")  # (a padded position may hold anything)
    buf = torch.full((40, 50), 3.0, device=DEV)
    got = g.embedding_grad(dy, tokens, 40, padding_idx=6, out=buf[:, 1:49])
    want, mag, count = _embedding_grad_want(dy.view(-1, 48), tokens.view(-1), 40, 1.0, 6)
    _close(got, want, (count + 2) * E32 * mag + E32 * want.abs())
    assert (got[6] == 0).all() and (buf[:, 0] == 3).all() and (buf[:, 49] == 3).all()
    # a layout without contiguous rows is written through a copy
    t = torch.empty((48, 40), device=DEV).t()
    assert torch.equal(g.embedding_grad(dy, tokens, 40, padding_idx=6, out=t), got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [2047, 2048, 2049, 3001, 4095, 4096, 4097])
@pytest.mark.parametrize("vocab,width,spread", [(1, 33, "even"), (61, 515, "zipf"), (9000, 131, "zipf"), (500, 64, "one")])
def test_embedding_grad_at_the_lists_sizes(n, vocab, width, spread, dtype):
    """Token counts at which the lists in LDS and the number of launches
    change, with all tokens in one row, one row per token and between."""
    gen = _gen(n + vocab)
    u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
    if spread == "even":
        tokens = (u * vocab).long().clamp_(max=vocab - 1)
    elif spread == "one":
        tokens = torch.where(u < 0.97, vocab // 2, (u * 31337).long() % vocab)
    else:
        tokens = ((torch.exp(u * math.log(vocab + 1.0)) - 1).long() * 7919 % vocab).clamp_(0, vocab - 1)
    dy = _randn(gen, (n, width), dtype)
    got = _twice(lambda: g.embedding_grad(dy, tokens, vocab))
    want, mag, count = _embedding_grad_want(dy, tokens, vocab, 1.0)
    _close(got, want, (count + 2) * E32 * mag + U[dtype] * want.abs() + TINY[dtype])
    assert (got[(count[:, 0] == 0)] == 0).all()


def test_embedding_grad_more_of_one_range_than_lds_lists():
    """Several rows of one workgroup's range with more tokens than its lists hold."""
    gen = _gen(9)
    n, vocab, width = 9000, 65536, 16
    tokens = torch.randint(128, 190, (n,), generator=gen, device=DEV)
    tokens[::17] = 40000
    dy = _randn(gen, (n, width), F16)
    got = _twice(lambda: g.embedding_grad(dy, tokens, vocab, dtype=F32))
    want, mag, count = _embedding_grad_want(dy, tokens, vocab, 1.0)
    _close(got, want, (count + 2) * E32 * mag + E32 * want.abs())


# --------------------------------------------------------------------------
# Layer norm
# --------------------------------------------------------------------------

# (rows, width): one vector to rows past what registers hold.
_NORMS = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 511), (4, 513), (300, 1027), (1, 4096), (7, 4097), (3, 8200), (2, 16384),
          (2, 16400), (2, 33000), (1031, 96)]
# Roundings of 2^-24 on the way of an output: fewer than 100 additions in a
# chain (a lane's columns, the exchanges, the waves), twice over for the
# variance and the products after it.
_K = 200


def _norm_want(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    y = xh * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean, rstd, xh


@pytest.mark.parametrize("dtype,pdtype", [(F16, F16), (BF16, BF16), (F32, F32), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("rows,width", _NORMS)
def test_layer_norm(rows, width, dtype, pdtype):
    gen = _gen(rows + width)
    x = _strided(_randn(gen, (rows, width), dtype, 1.5, 0.5), 3, 1)
    w, b = _randn(gen, (width,), pdtype, 0.2, 1.0), _randn(gen, (width,), pdtype, 0.3)
    y, mean, rstd = _twice(lambda: g.layer_norm(x, w, b))
    assert y.dtype == dtype and mean.dtype == rstd.dtype == F32 and mean.shape == (rows,)
    wy, wm, wr, _ = _norm_want(x, w, b, 1e-5)
    top = x.double().abs().amax(1, keepdim=True)
    _close(mean[:, None], wm, _K * E32 * top)
    # d rstd = rstd^3 / 2 d var, d var <= 2 |x| |dx|
    _close(rstd[:, None], wr, _K * E32 * (wr + wr**3 * top * top))
    tol = _K * E32 * ((wr + wr**3 * top * top) * 2 * top * w.double().abs() + b.double().abs())
    _close(y, wy, tol + U[dtype] * (wy.abs() + tol) + TINY[dtype])


def test_layer_norm_options():
    gen = _gen(1)
    x = _randn(gen, (2, 3, 130), BF16, 2.0)
    y, mean, rstd = g.layer_norm(x, eps=0.5)
    wy, wm, wr, _ = _norm_want(x.view(-1, 130), None, None, 0.5)
    assert y.shape == x.shape and mean.shape == (2, 3)
    _close(y.view(-1, 130), wy, U[BF16] * wy.abs() + 1e-4)
    b = _randn(gen, (130,), F32)
    y2 = g.layer_norm(x, bias=b, eps=0.5)[0]
    _close(y2.view(-1, 130), wy + b.double(), U[BF16] * (wy + b.double()).abs() + 1e-4)
    buf = torch.full((2, 3, 132), 5.0, dtype=BF16, device=DEV)
    out = g.layer_norm(x, eps=0.5, out=buf[..., 1:131])[0]
    assert torch.equal(out, y) and (buf[..., 0] == 5).all() and (buf[..., 131] == 5).all()
    assert g.layer_norm(x, eps=0.5, out=torch.empty((130, 3, 2), dtype=BF16, device=DEV).permute(2, 1, 0))[0].equal(y)
    # constant rows: no variance
    c, m, r = g.layer_norm(torch.full((3, 77), 4.0, device=DEV), eps=1e-5)
    assert (c == 0).all() and (m == 4).all()
    _close(r, torch.full((3,), 1e5**0.5, dtype=torch.float64, device=DEV), 1e-6 * 1e5**0.5)
    # a row that holds NaN or an infinity says so and leaves the others alone
    z = _randn(gen, (4, 300), F32)
    clean = g.layer_norm(z)[0]
    z[1, 5], z[2, 299] = float("nan"), float("inf")
    got = g.layer_norm(z)[0]
    assert got[1].isnan().all() and got[2].isnan().any()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])
    assert g.layer_norm(torch.empty((0, 40), device=DEV))[0].shape == (0, 40)
    # large offsets from zero do not cancel (two passes, not sums of squares)
    far = _randn(gen, (3, 4096), F32, 1.0, 3000.0)
    y, _, r = g.layer_norm(far)
    wy, _, wr, _ = _norm_want(far, None, None, 1e-5)
    _close(r[:, None], wr, 1e-3 * wr)


@pytest.mark.parametrize("dtype,pdtype", [(F16, F16), (BF16, BF16), (F32, F32), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("rows,width", _NORMS)
def test_layer_norm_grad(rows, width, dtype, pdtype):
    gen = _gen(rows * 3 + width)
    x = _strided(_randn(gen, (rows, width), dtype, 1.5, 0.5), 3, 1)
    dy = _strided(_randn(gen, (rows, width), dtype), 1, 2)
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
    chain = rows / 128 + 300
    big = rs * (x.double().abs() + mean.double().abs()[:, None])
    for got, wt, mag in ((dw, (dy.double() * xh).sum(0), (dy.double().abs() * (xh.abs() + big)).sum(0)),
                         (db, dy.double().sum(0), dy.double().abs().sum(0))):
        tol = chain * E32 * mag
        _close(got, wt, tol + U[pdtype] * (wt.abs() + tol) + TINY[pdtype])


def test_layer_norm_of_more_rows_than_one_grid_dimension():
    """More workgroups than 2^32 threads along one dimension of a grid have,
    and offsets past 2^31."""
    rows, width = (1 << 26) + 4100, 33
    x = torch.arange(rows, device=DEV).remainder_(251).to(F16)[:, None].repeat(1, width)
    x[:, ::2] += 3
    y, mean, rstd = g.layer_norm(x)
    m, var = 3 * 17 / 33, 9 * (17 / 33) * (16 / 33)
    want = torch.arange(rows, device=DEV).remainder_(251).double() + m
    assert ((mean.double() - want).abs() <= 40 * E32 * 256).all()
    del want
    r = 1 / math.sqrt(var + 1e-5)
    assert ((rstd.double() - r).abs() <= 200 * E32 * 256 * r).all()
    for c, v in ((0, (3 - m) * r), (31, -m * r), (32, (3 - m) * r)):
        assert ((y[:, c].double() - v).abs() <= U[F16] * abs(v) + 200 * E32 * 256 * r).all()


def test_layer_norm_grad_against_differences():
    """<dx, d> = d/dh of <dy, y(x + h d)>, and the same for the weight: central
    differences of the forward call itself in float32, summed in 64 bits."""
    gen = _gen(4)
    x, w, b = _randn(gen, (5, 300), F32), _randn(gen, (300,), F32, 0.2, 1.0), _randn(gen, (300,), F32)
    dy, d, dwt = _randn(gen, (5, 300), F32), _randn(gen, (5, 300), F32), _randn(gen, (300,), F32)
    _, mean, rstd = g.layer_norm(x, w, b)
    dx, dw, db = g.layer_norm_grad(dy, x, mean, rstd, w)
    h = 2.0**-6

    def f(xx, ww):
        return float((dy.double() * g.layer_norm(xx, ww, b)[0].double()).sum())

    # Rounding: 1500 terms of about 4 * 2^-24 each over 2 h; curvature: h^2 / 6
    # of a third derivative below 1500 * 30.
    tol = 1500 * 8 * E32 / (2 * h) + h * h / 6 * 1500 * 30 / 10
    assert abs((f(x + h * d, w) - f(x - h * d, w)) / (2 * h) - float((dx.double() * d.double()).sum())) < tol
    assert abs((f(x, w + h * dwt) - f(x, w - h * dwt)) / (2 * h) - float((dw.double() * dwt.double()).sum())) < tol
    _close(db, dy.double().sum(0), 5 * E32 * dy.double().abs().sum(0))


def test_layer_norm_grad_options():
    gen = _gen(6)
    x, dy = _randn(gen, (2, 4, 90), BF16), _randn(gen, (2, 4, 90), BF16)
    y, mean, rstd = g.layer_norm(x)
    dx, dw, db = g.layer_norm_grad(dy, x, mean, rstd)
    assert dx.shape == x.shape and dw.dtype == BF16
    one = torch.ones(90, dtype=BF16, device=DEV)
    for a, b in zip(g.layer_norm_grad(dy, x, mean, rstd, one), (dx, dw, db)):
        assert torch.equal(a, b)
    w32 = g.layer_norm_grad(dy, x, mean, rstd, one, param_dtype=F32)
    assert w32[1].dtype == F32 and torch.equal(w32[1].to(BF16), dw) and torch.equal(w32[0], dx)
    e = torch.empty((0, 90), device=DEV)
    s = torch.empty((0,), device=DEV)
    dx, dw, db = g.layer_norm_grad(e, e, s, s)
    assert dx.shape == (0, 90) and (dw == 0).all() and (db == 0).all()


# --------------------------------------------------------------------------
# Softmax cross entropy of a linear head
# --------------------------------------------------------------------------

_HEADS = [(1, 1, 1), (1, 2, 8), (2, 7, 3), (5, 300, 64), (31, 129, 70), (33, 257, 128), (64, 1000, 65), (130, 4097, 200),
          (257, 513, 264), (300, 20011, 96), (513, 1025, 1000), (16, 33000, 512), (1100, 8200, 320), (7, 9, 4100)]


def _head(t, v, d, dtype, seed, std=None, pad=0):
    gen = _gen(seed)
    w = _randn(gen, (v, d), dtype, std if std is not None else 2.0 / math.sqrt(d))
    x = _randn(gen, (t, d), dtype)
    y = torch.randint(0, v, (t,), generator=gen, device=DEV)
    if pad:
        x, w = _strided(x, pad, 1), _strided(w, pad, 3)
    return x, w, y


def _head_want(x, w, y, keep):
    """lse, loss, the logits' forward error bound, p - onehot, and p."""
    xd, wd = x.double(), w.double()
    xd = torch.where(keep[:, None], xd, 0.0)
    z = xd @ wd.t().contiguous()
    slack = (x.shape[1] + 2) * E32 * (xd.abs() @ wd.abs().t().contiguous()).amax(1)
    lse = torch.logsumexp(z, 1)
    loss = lse - z.gather(1, y[:, None])[:, 0]
    p = torch.exp(z - lse[:, None])
    gz = p.clone()
    gz.scatter_add_(1, y[:, None], torch.full_like(y[:, None], -1, dtype=torch.float64))
    return lse, loss, slack, gz, p


def _loss_tol(slack, lse):
    # two logits' sums, the sum of exponentials (each within 2^-21, fewer than
    # 200 additions in a chain) and the final additions
    return 2 * slack + 2.0**-21 + 200 * E32 + 4 * E32 * lse.abs()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("t,v,d", _HEADS)
def test_linear_cross_entropy(t, v, d, pad, dtype):
    x, w, y = _head(t, v, d, dtype, t + v + d, pad=pad)
    keep = torch.rand((t,), generator=_gen(t), device=DEV) < 0.8
    x[~keep] = float("nan")  # ignored rows may hold anything
    lse, loss, slack, _, _ = _head_want(x, w, y, keep)
    got = _twice(lambda: g.linear_cross_entropy(x, w, torch.where(keep, y, -100)))
    tol = _loss_tol(slack, lse)
    for a, b in zip(got, (loss, lse)):
        assert a.shape == (t,) and a.dtype == F32
        assert (a[~keep] == 0).all()
        _close(a[keep], b[keep], tol[keep])


def _grad_tols(x, w, gz, p, slack, keep, factor, dtype):
    """Bounds of dx and dw.  A probability carries its logit's and the lse's
    error, the exponentials' (2^-20), their f16 form relative to a maximum of 1
    (2^-11 of the value, 2^-25 near zero) and the rounding to the operands'
    type; the products' sums and the result's rounding come on top."""
    rel = (2 * slack[:, None] + 2.0**-19 + 2.0**-11) * (1 + U[dtype])
    eps = rel * p + U[dtype] * gz.abs() + 2.0**-24
    eps = torch.where(keep[:, None], eps, 0.0)
    gz = torch.where(keep[:, None], gz, 0.0)
    xd, wd = torch.where(keep[:, None], x.double(), 0.0), w.double()
    dx = factor * (gz @ wd)
    dw = factor * (gz.t().contiguous() @ xd)
    tx = factor * (((eps + (w.shape[0] + 40) * E32 * gz.abs())) @ wd.abs())
    tw = factor * ((eps + (x.shape[0] + 4) * E32 * gz.abs()).t().contiguous() @ xd.abs())
    return (dx, tx + U[dtype] * (dx.abs() + tx) + TINY[dtype]), (dw, tw + U[dtype] * (dw.abs() + tw) + TINY[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("t,v,d", _HEADS)
def test_linear_cross_entropy_grad(t, v, d, pad, dtype):
    x, w, y = _head(t, v, d, dtype, 2 * t + v + d, pad=pad)
    keep = torch.rand((t,), generator=_gen(t), device=DEV) < (0.75 if t > 1 else 2)
    x[~keep] = float("nan")
    count = max(1, int(keep.sum()))
    lse, loss, slack, gz, p = _head_want(x, w, y, keep)
    targets = torch.where(keep, y, 2**31 - 1).int()
    for reduction, share in (("mean", 1.0 / count), ("sum", 1.0)):
        got = _twice(lambda: g.linear_cross_entropy_grad(x, w, targets, ignore_index=2**31 - 1, reduction=reduction,
                                                         grad_scale=8.0))
        assert got[0].shape == () and got[1].dtype == got[2].dtype == dtype
        tol = (_loss_tol(slack, lse)[keep].sum() + (t / 1024 + 30) * E32 * loss[keep].abs().sum()) * share
        assert abs(float(got[0]) - float(loss[keep].sum()) * share) <= float(tol) + 1e-30
        (dx, tx), (dw, tw) = _grad_tols(x, w, gz, p, slack, keep, 8.0 * share, dtype)
        _close(got[1], dx, tx)
        _close(got[2], dw, tw)
        assert (got[1][~keep] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_peaked_and_shifted_logits(dtype):
    """Logits of some hundreds, a token whose target is certain, one whose
    target is hopeless, rows of equal logits."""
    t, v, d = 70, 700, 64
    gen = _gen(3)
    w = _randn(gen, (v, d), dtype)
    x = _randn(gen, (t, d), dtype, 12.0)
    x[3] = w[5] * 20
    x[4] = w[5] * 20
    x[5] = 0
    y = torch.randint(0, v, (t,), generator=gen, device=DEV)
    y[3], y[4] = 5, 6
    keep = torch.ones((t,), dtype=torch.bool, device=DEV)
    lse, loss, slack, gz, p = _head_want(x, w, y, keep)
    got_loss, got_lse = g.linear_cross_entropy(x, w, y)
    tol = _loss_tol(slack, lse)
    _close(got_loss, loss, tol)
    _close(got_lse, lse, tol)
    total, gx, gw = g.linear_cross_entropy_grad(x, w, y, reduction="sum")
    (dx, tx), (dw, tw) = _grad_tols(x, w, gz, p, slack, keep, 1.0, dtype)
    _close(gx, dx, tx)
    _close(gw, dw, tw)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nothing_counts_and_empty(dtype):
    x, w, y = _head(9, 50, 24, dtype, 0)
    loss, dx, dw = g.linear_cross_entropy_grad(x, w, torch.full_like(y, -100))
    assert float(loss) == 0 and (dx == 0).all() and (dw == 0).all()
    a, b = g.linear_cross_entropy(x, w, torch.full_like(y, -100))
    assert (a == 0).all() and (b == 0).all()
    loss, dx, dw = g.linear_cross_entropy_grad(x[:0], w, y[:0])
    assert float(loss) == 0 and dx.shape == (0, 24) and (dw == 0).all()
    assert g.linear_cross_entropy(x[:0], w, y[:0])[0].shape == (0,)
    x3 = x.view(3, 3, 24)
    a3, _ = g.linear_cross_entropy(x3, w, y.view(3, 3))
    assert torch.equal(a3.view(-1), g.linear_cross_entropy(x, w, y)[0])


def test_targets_outside_and_bad_rows():
    x, w, y = _head(6, 300, 40, BF16, 1)
    clean, _ = g.linear_cross_entropy(x, w, y)
    y2 = y.clone()
    y2[1], y2[4] = 300, -7
    loss, lse = g.linear_cross_entropy(x, w, y2)
    assert loss[1].isnan() and loss[4].isnan() and lse.isfinite().all()
    ok = [0, 2, 3, 5]
    assert torch.equal(loss[ok], clean[ok])
    x[2, 3] = float("nan")
    loss, _ = g.linear_cross_entropy(x, w, y)
    assert loss[2].isnan() and torch.equal(loss[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]])
    # a vocabulary row whose logit is -inf has no weight in the softmax
    x = x.abs() + 0.5
    x[2, 3] = 1.0
    w[7] = float("-inf")
    y[y == 7] = 8
    loss, lse = g.linear_cross_entropy(x, w, y)
    rest = [i for i in range(300) if i != 7]
    want, _ = g.linear_cross_entropy(x, w[rest], torch.where(y > 7, y - 1, y))
    _close(loss, want.double(), 1e-5 * (1 + want.double().abs()))


def test_gradient_against_differences():
    """<dx, e> and <dw, e> against central differences of the forward call.
    Inputs are multiples of 2^-7 and the step a power of two, so the moved
    ones are exact in float16."""
    gen = _gen(8)
    t, v, d = 40, 333, 32
    x = (torch.randint(-128, 129, (t, d), generator=gen, device=DEV) / 128.0).half()
    w = (torch.randint(-64, 65, (v, d), generator=gen, device=DEV) / 128.0).half()
    y = torch.randint(0, v, (t,), generator=gen, device=DEV)
    ex = torch.randint(-1, 2, (t, d), generator=gen, device=DEV).half()
    ew = torch.randint(-1, 2, (v, d), generator=gen, device=DEV).half()
    h = 2.0**-5
    _, dx, dw = g.linear_cross_entropy_grad(x, w, y, reduction="sum")

    def f(xx, ww):
        return float(g.linear_cross_entropy(xx, ww, y)[0].double().sum())

    for a, b, grad, e, other in (((x + h * ex, w), (x - h * ex, w), dx, ex, w.double().abs()),
                                 ((x, w + h * ew), (x, w - h * ew), dw, ew, x.double().abs())):
        assert torch.equal((a[0] - b[0]), 2 * h * ex) or torch.equal((a[1] - b[1]), 2 * h * ew)
        slope = (f(*a) - f(*b)) / (2 * h)
        want = float((grad.double() * e.double()).sum())
        # A logit moves by at most `move` per unit of h; a token's third
        # derivative is a third central moment, below (2 move)^3 / 10.
        move = float((e.double().abs() @ other.t().contiguous()).amax())
        curve = h * h / 6 * t * (2 * move) ** 3 / 10
        noise = t * 2.0**-19 / h
        rounding = 3 * U[F16] * float((grad.double().abs() * e.double().abs()).sum())
        assert abs(slope - want) <= curve + noise + rounding, (slope, want, curve, noise, rounding)


@pytest.mark.parametrize("ignored", [50, 5, 2])
def test_more_tokens_than_one_piece(ignored):
    """More tokens than one piece holds (1 GiB of probabilities, 4096 tokens
    here): a second piece with tokens, and one that is left without any."""
    t, v, d = 4500, 131072, 64
    x, w, y = _head(t, v, d, BF16, 11, std=0.2)
    keep = torch.ones((t,), dtype=torch.bool, device=DEV)
    keep[::ignored] = False
    lse, loss, slack, gz, p = _head_want(x, w, y, keep)
    got = g.linear_cross_entropy_grad(x, w, torch.where(keep, y, -100), reduction="sum")
    tol = _loss_tol(slack, lse)[keep].sum() + (t / 1024 + 30) * E32 * loss[keep].abs().sum()
    assert abs(float(got[0]) - float(loss[keep].sum())) <= float(tol)
    (dx, tx), (dw, tw) = _grad_tols(x, w, gz, p, slack, keep, 1.0, BF16)
    _close(got[1], dx, tx)
    _close(got[2], dw, tw)


@pytest.mark.parametrize("t,v,d,ignored", [(65537, 5, 8, 3), (200003, 70, 16, 2), ((1 << 24) + 5000, 3, 8, 4)])
def test_many_tokens(t, v, d, ignored):
    """More tokens than one launch counts in one go, and than one piece has."""
    x, w, y = _head(t, v, d, BF16, 12)
    keep = torch.ones((t,), dtype=torch.bool, device=DEV)
    keep[::ignored] = False
    keep[70000 : min(t, 140000)] = False
    lse, loss, slack, gz, p = _head_want(x, w, y, keep)
    targets = torch.where(keep, y, -100)
    got = g.linear_cross_entropy(x, w, targets)
    for a, want in zip(got, (loss, lse)):
        _close(a[keep], want[keep], _loss_tol(slack, lse)[keep])
        assert (a[~keep] == 0).all()
    got = g.linear_cross_entropy_grad(x, w, targets, reduction="sum")
    tol = _loss_tol(slack, lse)[keep].sum() + (t / 1024 + 30) * E32 * loss[keep].abs().sum()
    assert abs(float(got[0]) - float(loss[keep].sum())) <= float(tol)
    (dx, tx), (dw, tw) = _grad_tols(x, w, gz, p, slack, keep, 1.0, BF16)
    _close(got[1], dx, tx)
    _close(got[2], dw, tw)


# --------------------------------------------------------------------------
# Streams, graphs, refusals
# --------------------------------------------------------------------------


def _step(x, table, tokens, w, b, y, dy):
    e = g.embedding(tokens, table, scale=2.0)
    h, mean, rstd = g.layer_norm(e, w, b)
    loss, dh, dhead = g.linear_cross_entropy_grad(h, table, y)
    dx, dw, db = g.layer_norm_grad(dh, e, mean, rstd, w)
    return loss, dhead, g.embedding_grad(dx, tokens, table.shape[0], scale=2.0), dw, db


def _step_args(seed, t=200, v=700, d=72):
    gen = _gen(seed)
    return (None, _randn(gen, (v, d), BF16, 0.3), torch.randint(0, v, (t,), generator=gen, device=DEV),
            _randn(gen, (d,), BF16, 0.1, 1.0), _randn(gen, (d,), BF16, 0.1),
            torch.randint(0, v, (t,), generator=gen, device=DEV), None)


def test_on_other_streams():
    args = [_step_args(s) for s in range(3)]
    want = [_step(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            got.append(_step(*a))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_captured_into_a_graph():
    args = _step_args(7)
    _step(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*args)
    for seed in (1, 2, 3):
        new = _step_args(seed)
        for a, b in zip(args, new):
            if a is not None:
                a.copy_(b)
        want = _step(*args)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), seed


def test_refusals_on_device_tensors():
    x = torch.zeros((4, 8), dtype=BF16, device=DEV)
    ids = torch.zeros((4,), dtype=torch.int64, device=DEV)
    for call, match in (
            (lambda: g.embedding(ids.float(), x), "int32 or int64"),
            (lambda: g.embedding(ids, x[0]), "2-D"),
            (lambda: g.embedding(ids, x.double()), "float64"),
            (lambda: g.embedding(ids.cpu(), x), "GPU"),
            (lambda: g.embedding(ids, x, out=torch.zeros((4, 9), dtype=BF16, device=DEV)), "out shape"),
            (lambda: g.embedding(ids, x, out=torch.zeros((4, 8), device=DEV)), "out must be bfloat16"),
            (lambda: g.embedding_grad(x, ids[:3], 5), "does not match tokens"),
            (lambda: g.embedding_grad(x, ids, -1), "negative"),
            (lambda: g.embedding_grad(x, ids, 5, padding_idx=5), "outside the vocabulary"),
            (lambda: g.embedding_grad(x, ids, 5, dtype=F16), "bfloat16 or float32"),
            (lambda: g.layer_norm(x, torch.ones((7,), dtype=BF16, device=DEV)), "width 8"),
            (lambda: g.layer_norm(x, torch.ones((8,), dtype=F16, device=DEV)), "bfloat16 or float32"),
            (lambda: g.layer_norm(x, torch.ones((8,), dtype=BF16, device=DEV), torch.ones((8,), device=DEV)), "one type"),
            (lambda: g.layer_norm(x[:, :0]), "without elements"),
            (lambda: g.layer_norm(x.double()), "float64"),
            (lambda: g.layer_norm_grad(x, x, ids.float()[:3], ids.float()), "4 float32 values"),
            (lambda: g.layer_norm_grad(x.half(), x, ids.float(), ids.float()), "as x"),
            (lambda: g.layer_norm_grad(x[:2], x, ids.float(), ids.float()), "does not match x"),
            (lambda: g.linear_cross_entropy(x.float(), x.float(), ids), "float16 or bfloat16"),
            (lambda: g.linear_cross_entropy(x, x.half(), ids), "one type"),
            (lambda: g.linear_cross_entropy(x, x[:, :7], ids), "do not match"),
            (lambda: g.linear_cross_entropy(x, x, ids[:3]), "targets shape"),
            (lambda: g.linear_cross_entropy(x, x[:0], ids), "no vocabulary"),
            (lambda: g.linear_cross_entropy(x, x, ids.float()), "int32 or int64"),
            (lambda: g.linear_cross_entropy_grad(x, x, ids, reduction="max"), "reduction"),
            (lambda: g.linear_cross_entropy_grad(x, 3, ids), "torch tensor")):
        with pytest.raises(LaunchError, match=match):
            call()
