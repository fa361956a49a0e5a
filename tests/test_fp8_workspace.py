"""The scratch of the 8-bit product, on the host: its query plans no call that
the product refuses, whatever its sizes, and the product takes no scratch that is
missing, short or misaligned."""

from __future__ import annotations

import re

import pytest

pytest.importorskip("torch")

from hc.gfx950 import _native

BF16, F32, E4M3 = _native.HCG_BF16, _native.HCG_F32, _native.HCG_E4M3
P = 0x1000  # any non-null, aligned pointer: a rejected call never reads it
FORMS = [v for v in _native.FP8_ALGOS.values()]


def _need(algo, tokens, outputs, inputs, x=P, xs_row=1, out=BF16):
    return _native.load().hcg_linear_fp8_workspace(algo, tokens, outputs, inputs, x, inputs, P, inputs, F32, xs_row, 1, P, 1,
                                                   1, out)


def _call(algo, tokens, outputs, inputs, work, size, x=P, xs_row=1, out=BF16):
    rc = _native.load().hcg_linear_fp8(algo, E4M3, x, inputs, tokens, P, inputs, outputs, inputs, F32, P, xs_row, 3, 1, P, 1,
                                       1, out, P, outputs, work, size, None)
    return rc, _native.last_error(_native.load())


@pytest.mark.parametrize("algo", FORMS)
@pytest.mark.parametrize("tokens,outputs,inputs", [
    (1, 1, 4000000), (1, 1, 1 << 31), (1, 1, 1 << 32), (3, 5, 1 << 36), (3, 5, (1 << 62) + 1), (1 << 26, 5, 128),
    (1 << 40, 5, 128), (3, 1 << 26, 128), (3, 1 << 62, 1 << 40), (-1, 5, 128), (3, -1, 128), (3, 5, -128)])
def test_sizes_out_of_range_need_none(tokens, outputs, inputs, algo):
    assert _need(algo, tokens, outputs, inputs) == 0
    rc, text = _call(algo, tokens, outputs, inputs, P, 1 << 40)
    assert rc == _native.HCG_EINVAL and "out of range" in text


@pytest.mark.parametrize("algo", [-1, 5, 99, 255, 256, 512, 256 * 17 + 3, (1 << 31) - 1, -(1 << 31)])
def test_unknown_forms_need_none(algo):
    assert _need(algo, 64, 512, 8192) == 0
    rc, text = _call(algo, 64, 512, 8192, P, 1 << 40)
    assert rc == _native.HCG_EINVAL and f"unknown algo {algo}" in text


def test_too_many_tiles_need_none():
    """Sizes in range whose tiles no launch holds."""
    many = (1 << 26) - 1
    for algo in (0, 2, 3, 4):
        assert _need(algo, many, many, 128, out=F32) == 0
        rc, text = _call(algo, many, many, 128, P, 1 << 40, out=F32)
        assert rc == _native.HCG_EINVAL and "out of range" in text


# Split sums; rows at no multiple of 16 bytes; scales of strided rows.
@pytest.mark.parametrize("algo,change", [(3 + 256 * 4, {}), (1 + 256 * 3, {}), (2, {"x": P + 1}), (4, {"xs_row": 3})])
def test_scratch_is_asked_for(algo, change):
    need = _need(algo, 64, 512, 8192, **change)
    assert need > 0
    for work, size in ((None, need), (P, need - 1), (P, 0), (P + 16, need)):
        rc, text = _call(algo, 64, 512, 8192, work, size, **change)
        assert rc == _native.HCG_EINVAL and re.search(rf"workspace of {size} bytes, {need} needed", text)
