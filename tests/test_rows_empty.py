"""Rows without elements keep their number, whatever the dimensions in front: a
product over no inputs is refused and a matrix of no columns keeps its shape when it
is quantised."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc._errors import LaunchError  # noqa: E402
from hc.gfx950.lm import _rows  # noqa: E402

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("shape,rows", [((0,), 1), ((6, 0), 6), ((2, 3, 0), 6), ((2, 0, 0), 0), ((2, 1, 3, 0), 6),
                                        ((0, 3, 5), 0), ((2, 0, 5), 0), ((2, 3, 5), 6), ((5,), 1)])
def test_number_of_rows(shape, rows):
    assert _rows(torch.empty(shape), "x").shape == (rows, shape[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(6,), (2, 3), (1, 2, 3), ()])
def test_product_over_no_inputs(lead):
    x, s = torch.empty((*lead, 0), dtype=E4M3, device=DEV), torch.empty((*lead, 0), device=DEV)
    w, ws = torch.empty((40, 0), dtype=E4M3, device=DEV), torch.empty((1, 0), device=DEV)
    with pytest.raises(LaunchError, match="no inputs"):
        g.linear_fp8(x, s, w, ws)
    with pytest.raises(LaunchError, match="no inputs"):
        g.linear_fp8(x, s, w, ws, out=torch.empty((*lead, 40), dtype=torch.bfloat16, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(6,), (2, 3), (1, 2, 3)])
def test_quantising_no_columns(lead):
    x = torch.empty((*lead, 0), dtype=torch.bfloat16, device=DEV)
    q, s = g.quantize_fp8(x)
    assert q.shape == x.shape and s.shape == (*lead, 0)
    assert g.quantize_fp8(x, block="tile")[1].shape == (1, 0)
    q, s = g.quantize_fp8(x, transpose=True)
    assert q.shape == (0, 6) and s.shape == (0, 1)
    assert g.quantize_fp8(x, transpose=True, block="tile")[1].shape == (0, 1)


@pytest.mark.gpu
def test_other_operators_of_no_columns():
    tokens = torch.tensor([[0, 1, 2], [2, 1, 0]], device=DEV)
    dy = torch.empty((2, 3, 0), device=DEV)
    assert g.embedding_grad(dy, tokens, 7).shape == (7, 0)
    assert g.embedding_grad(dy, tokens, 7, padding_idx=1).shape == (7, 0)
    for call in (lambda: g.layer_norm(dy), lambda: g.rms_norm(dy), lambda: g.rms_norm_fp8(dy)):
        with pytest.raises(LaunchError, match="without elements"):
            call()
