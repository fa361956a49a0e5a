"""The 8-bit product's operands where they are hard, for every type of result:
NaNs, infinities and scales that are none, rows that end inside 16 bytes with
NaN behind them, the smallest and largest exponents as scales.

Elements are whole numbers up to 4 and scales powers of two, so that every sum is
a float32 number, and no product is below 2^-13 of the largest, 16, of its
neighbours: results of every type are the rounded sums, bit for bit."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
FORMS = ["stream", "stream/3", "256x256", "256x256/3", "128x128", "128x128/2", "128x64", "128x64/3", "auto"]
RESULTS = [BF16, F16, F32]
OPERANDS = [(E4M3, True, F32), (E5M2, False, F32), (E4M3, False, E8M0), (E5M2, True, E8M0)]


def _blocks(n):
    return -(-n // 128)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _operands(seed, tokens, outputs, inputs, x_dtype, tile, scale_dtype):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def whole(rows, dtype):
        return torch.randint(-4, 5, (rows, inputs), generator=gen, device=DEV).float().to(dtype)

    def scales(rows):
        return torch.exp2(torch.randint(-1, 2, (rows, _blocks(inputs)), generator=gen, device=DEV).float()).to(scale_dtype)

    return whole(tokens, x_dtype), scales(tokens), whole(outputs, E4M3), scales(_blocks(outputs) if tile else outputs)


def _want(x, sx, w, sw, tile):
    def stands(q, s, high):
        rows, cols = (torch.arange(n, device=DEV) for n in q.shape)
        return q.double() * s.double()[rows // high][:, cols // 128]

    return stands(x, sx, 1) @ stands(w, sw, 128 if tile else 1).t().contiguous()


def _behind(t, pad, offset=0):
    """t in rows `pad` bytes longer that start `offset` bytes past a multiple of 256, NaN in between."""
    rows, cols = t.shape
    buf = torch.full((offset + rows * (cols + pad) + 16,), 0x7F, dtype=torch.uint8, device=DEV)
    view = buf[offset : offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_(_bytes(t))
    return view.view(t.dtype)


@pytest.mark.parametrize("result", RESULTS)
@pytest.mark.parametrize("algo", FORMS)
@pytest.mark.parametrize("x_dtype,tile,scale_dtype", OPERANDS)
@pytest.mark.parametrize("tokens,outputs,inputs", [(1, 1, 1), (3, 5, 7), (17, 40, 131), (65, 130, 1000), (129, 257, 1027),
                                                   (300, 515, 300), (64, 128, 2047)])
def test_rows_with_nan_behind_them(tokens, outputs, inputs, x_dtype, tile, scale_dtype, algo, result):
    x, sx, w, sw = _operands(inputs, tokens, outputs, inputs, x_dtype, tile, scale_dtype)
    want = _want(x, sx, w, sw, tile).float().to(result)
    # read where they lie: whole 16 bytes from row to row, the last ones NaN from the row's end on
    got = g.linear_fp8(_behind(x, 16 - inputs % 16), sx, _behind(w, 32 - inputs % 16), sw, out_dtype=result, algo=algo)
    assert torch.equal(got, want)
    # at any address: copied by the tiled forms
    got = g.linear_fp8(_behind(x, 5, 3), sx, _behind(w, 7, 1), sw, out_dtype=result, algo=algo)
    assert torch.equal(got, want)


@pytest.mark.parametrize("result", RESULTS)
@pytest.mark.parametrize("algo", FORMS)
@pytest.mark.parametrize("x_dtype,tile,scale_dtype", OPERANDS)
def test_nan_stays_where_it_is(x_dtype, tile, scale_dtype, algo, result):
    """A NaN of a token's row, a weight's row or a scale reaches the results of
    that row, or tile, and no other, and so does an infinity."""
    tokens, outputs, inputs = 270, 300, 300
    x, sx, w, sw = _operands(9, tokens, outputs, inputs, x_dtype, tile, scale_dtype)
    want = _want(x, sx, w, sw, tile).float().to(result)
    xb, wb = _bytes(x).clone(), _bytes(w).clone()
    xb[3, 299] = xb[269, 0] = 0x7F
    wb[149, 131] = wb[299, 64] = 0xFF
    if x_dtype is E5M2:
        xb[68, 0], xb[200, 290] = 0x7C, 0xFC  # infinities
    sx, sw = sx.clone(), sw.clone()
    sx[11, 1] = sx[258, 2] = float("nan")
    sw[1 if tile else 7, 2] = float("nan")
    got = g.linear_fp8(xb.view(x_dtype), sx, wb.view(E4M3), sw, out_dtype=result, algo=algo)
    bad = torch.zeros((tokens, outputs), dtype=torch.bool, device=DEV)
    bad[[3, 11, 258, 269]] = True
    bad[:, [149, 299]] = True
    bad[:, slice(128, 256) if tile else 7] = True
    assert got[bad].isnan().all()
    if x_dtype is E5M2:
        assert not got[[68, 200]].isfinite().any()
        bad[[68, 200]] = True
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("result", RESULTS)
@pytest.mark.parametrize("algo", FORMS)
@pytest.mark.parametrize("x_dtype", [E4M3, E5M2])
@pytest.mark.parametrize("tile", [True, False])
def test_exponents_at_the_ends(tile, x_dtype, algo, result):
    """e8m0 bytes 0 (2^-127), 254 (2^127) and 255 (NaN): blocks whose two scales
    multiply to 1, 2 and 1/2."""
    tokens, outputs, inputs = 140, 260, 700
    x, sx, w, sw = _operands(10, tokens, outputs, inputs, x_dtype, tile, E8M0)
    sx = torch.tensor([0, 254, 127, 254, 0, 1], dtype=torch.uint8, device=DEV).expand(tokens, 6).contiguous()
    sw = torch.tensor([254, 0, 127, 1, 253, 254], dtype=torch.uint8, device=DEV).expand(sw.shape[0], 6).contiguous()
    want = _want(x, sx.view(E8M0), w, sw.view(E8M0), tile).float().to(result)
    sx[5, 5] = sx[139, 0] = 255
    sw[2 if tile else 9, 3] = 255
    got = g.linear_fp8(x, sx.view(E8M0), w, sw.view(E8M0), out_dtype=result, algo=algo)
    bad = torch.zeros((tokens, outputs), dtype=torch.bool, device=DEV)
    bad[[5, 139]] = True
    bad[:, slice(256, 260) if tile else 9] = True
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], want[~bad])
