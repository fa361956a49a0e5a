"""The language-model operators refuse parameters, statistics and losses that
are not aligned to their elements, on the host before any launch."""

from __future__ import annotations

import re

import pytest

pytest.importorskip("torch")

from hc.gfx950 import _native

BF16, F32 = _native.HCG_BF16, _native.HCG_F32
P = 0x1000  # any non-null, aligned pointer: a rejected call never reads it


def _refused(rc):
    assert rc == _native.HCG_EINVAL
    assert re.search("aligned", _native.last_error(_native.load()))


@pytest.mark.parametrize("name,by,pdtype", [("weight", 1, BF16), ("bias", 1, BF16), ("weight", 2, F32), ("bias", 2, F32),
                                            ("mean", 2, BF16), ("rstd", 1, BF16)])
def test_layer_norm(name, by, pdtype):
    a = dict(dtype=BF16, x=P, ldx=8, rows=3, width=8, pdtype=pdtype, weight=P, bias=P, eps=1e-5, y=P, ldy=8, mean=P,
             rstd=P, stream=None)
    a[name] += by
    _refused(_native.load().hcg_layer_norm(*a.values()))


@pytest.mark.parametrize("name,by,pdtype", [("weight", 1, BF16), ("dw", 1, BF16), ("db", 1, BF16), ("weight", 2, F32),
                                            ("dw", 2, F32), ("db", 2, F32), ("mean", 2, BF16), ("rstd", 2, BF16)])
def test_layer_norm_grad(name, by, pdtype):
    a = dict(dtype=BF16, dy=P, lddy=8, x=P, ldx=8, rows=3, width=8, mean=P, rstd=P, pdtype=pdtype, weight=P, dx=P,
             lddx=8, dw=P, db=P, ws=P, ws_bytes=1 << 30, stream=None)
    a[name] += by
    _refused(_native.load().hcg_layer_norm_grad(*a.values()))


@pytest.mark.parametrize("name", ["loss", "lse"])
def test_linear_cross_entropy(name):
    a = dict(dtype=BF16, x=P, ldx=8, tokens=3, weight=P, ldw=8, vocab=5, width=8, id_bytes=8, targets=P, ignore=-100,
             loss=P, lse=P, ws=P, ws_bytes=1 << 30, stream=None)
    a[name] += 2
    _refused(_native.load().hcg_linear_cross_entropy(*a.values()))


def test_linear_cross_entropy_grad():
    a = dict(dtype=BF16, x=P, ldx=8, tokens=3, weight=P, ldw=8, vocab=5, width=8, id_bytes=8, targets=P, ignore=-100,
             mean=1, scale=1.0, loss=P + 2, dx=P, lddx=8, dw=P, lddw=8, ws=P, ws_bytes=1 << 30, stream=None)
    _refused(_native.load().hcg_linear_cross_entropy_grad(*a.values()))
