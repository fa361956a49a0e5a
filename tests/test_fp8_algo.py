"""The names of the 8-bit product's forms: what is no form, or no number of
parts up to 16 in plain digits, is refused."""

from __future__ import annotations

import pytest

pytest.importorskip("torch")

from hc._errors import LaunchError
from hc.gfx950 import _native
from hc.gfx950.fp8 import _algo_number


def test_forms():
    for name, number in _native.FP8_ALGOS.items():
        assert _algo_number(name) == number
        if name != "auto":
            assert _algo_number(f"{name}/0") == number
            for parts in (1, 4, 16):
                assert _algo_number(f"{name}/{parts}") == number + _native.FP8_SPLITS * parts


@pytest.mark.parametrize("algo", ["", "best", "/4", "auto/4", "stream/17", "stream/-1", "stream/+1",
                                  "stream/ 1", "stream/1/1", "128x128/²", "128x128/٤", "128x64/4.0",
                                  f"stream/{1 << 24}", f"stream/{(1 << 24) + 2}", f"stream/{1 << 64}", "stream/" + "9" * 5000, None, 1])
def test_what_is_none_is_refused(algo):
    with pytest.raises(LaunchError, match="unknown algo"):
        _algo_number(algo)
