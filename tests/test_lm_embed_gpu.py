"""hc.gfx950.embedding on tables with strided columns."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402

from .test_lm_gpu import BF16, DEV, F16, F32, _gen, _randn  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_lookup_in_a_table_of_strided_columns(dtype):
    table = _randn(_gen(1), (40, 90), dtype)[::2, ::3]
    tokens = torch.tensor([3, 19, 20, 0, -1, 3], device=DEV)
    out = g.embedding(tokens, table, scale=0.75)
    known = torch.tensor([True, True, False, True, False, True], device=DEV)
    assert torch.equal(out[known], (table[tokens[known]].float() * 0.75).to(dtype))
    assert out[~known].isnan().all()
