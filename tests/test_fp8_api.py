"""The 8-bit linear layers and the root-mean-square norm without a GPU: the
library exports what include/hcg_fp8.h declares, bad arguments are rejected on
the host before any launch, and the Python entry points refuse tensors that are
not on a GPU."""

from __future__ import annotations

import os
import re

import pytest

import hc.gfx950 as g
from hc._errors import LaunchError
from hc.gfx950 import _native

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32 = _native.HCG_F16, _native.HCG_BF16, _native.HCG_F32
E4M3, E5M2, E8M0 = _native.HCG_E4M3, _native.HCG_E5M2, _native.HCG_E8M0
P = 0x1000  # any non-null, aligned pointer: a rejected call never reads it


def test_header_and_library_agree():
    text = open(os.path.join(ROOT, "include", "hcg_fp8.h")).read()
    declared = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(hcg_\w+)\s*\(", text, re.M)))
    assert declared == sorted(_native.FP8_EXPORTS)
    lib = _native.load()
    for name in declared:
        assert hasattr(lib, name), name
    for name, value in (("HCG_E4M3", E4M3), ("HCG_E5M2", E5M2), ("HCG_E8M0", E8M0), ("HCG_FP8_BLOCK", _native.FP8_BLOCK)):
        assert re.search(rf"#define {name} (\d+)", text).group(1) == str(value)
    for name, value in _native.FP8_ALGOS.items():
        assert re.search(rf"(?i)#define HCG_FP8_{name} (\d+)", text).group(1) == str(value)


def _refused(rc, match):
    assert rc == _native.HCG_EINVAL
    assert re.search(match, _native.last_error(_native.load())), _native.last_error(_native.load())


_ROWS = [({"dtype": 9}, "dtype 9"), ({"pdtype": F16}, "type or float32"), ({"rdtype": F16}, "type or float32"),
         ({"rows": -1}, "out of range"), ({"rows": 1 << 31}, "out of range"), ({"width": (1 << 30) + 1}, "out of range"),
         ({"width": 0}, "without elements"), ({"x": None}, "null"), ({"h": None}, "null"), ({"ldx": 7}, "stride"),
         ({"ldr": 7}, "stride"), ({"ldh": 7}, "stride"), ({"x": P + 1}, "aligned"), ({"residual": P + 1}, "aligned"),
         ({"h": P + 1}, "aligned"), ({"weight": P + 1}, "aligned"), ({"rstd": P + 2}, "aligned")]


@pytest.mark.parametrize("change,match", _ROWS + [({"y": None}, "null"), ({"ldy": 7}, "stride"), ({"y": P + 1}, "aligned")])
def test_rms_norm_arguments(change, match):
    a = dict(dtype=BF16, x=P, ldx=8, rows=3, width=8, rdtype=BF16, residual=P, ldr=8, pdtype=BF16, weight=P, eps=1e-6, y=P,
             ldy=8, h=P, ldh=8, rstd=P, stream=None)
    a.update(change)
    _refused(_native.load().hcg_rms_norm(*a.values()), match)


@pytest.mark.parametrize("change,match", _ROWS + [
    ({"qdtype": F16}, "q's type 0"), ({"sdtype": BF16}, "scales of type 1"), ({"q": None}, "null"), ({"scale": None}, "null"),
    ({"ldq": 7}, "stride"), ({"scale": P + 2}, "scales must be aligned")])
def test_rms_norm_fp8_arguments(change, match):
    a = dict(dtype=BF16, x=P, ldx=8, rows=3, width=8, rdtype=BF16, residual=P, ldr=8, pdtype=BF16, weight=P, eps=1e-6,
             qdtype=E4M3, q=P, ldq=8, sdtype=F32, scale=P, srow=1, sblock=3, h=P, ldh=8, rstd=P, stream=None)
    a.update(change)
    _refused(_native.load().hcg_rms_norm_fp8(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"dtype": 9}, "dtype 9"), ({"pdtype": F16}, "type or float32"), ({"hdtype": F16}, "type or float32"),
    ({"rows": 1 << 31}, "out of range"), ({"width": 0}, "without elements"), ({"dy": None}, "null"), ({"h": None}, "null"),
    ({"rstd": None}, "null"), ({"dh": None}, "null"), ({"lddy": 7}, "stride"), ({"ldh": 7}, "stride"), ({"lddr": 7}, "stride"),
    ({"lddh": 7}, "stride"), ({"dy": P + 1}, "aligned"), ({"h": P + 1}, "aligned"), ({"dres": P + 1}, "aligned"),
    ({"dh": P + 1}, "aligned"), ({"dw": P + 1}, "aligned"), ({"rstd": P + 2}, "aligned"), ({"ws": None}, "workspace"),
    ({"ws_bytes": 8}, "workspace of 8"), ({"ws": P + 16}, "workspace")])
def test_rms_norm_grad_arguments(change, match):
    a = dict(dtype=BF16, dy=P, lddy=8, hdtype=BF16, h=P, ldh=8, rows=3, width=8, rstd=P, pdtype=BF16, weight=P, dres=P,
             lddr=8, dh=P, lddh=8, dw=P, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(change)
    _refused(_native.load().hcg_rms_norm_grad(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"dtype": E4M3}, "dtype 3"), ({"qdtype": F32}, "q's type 2"), ({"sdtype": F16}, "scales of type 0"),
    ({"rows": -1}, "out of range"), ({"cols": 1 << 31}, "out of range"),
    ({"rows": (1 << 31) - 1, "cols": (1 << 31) - 1, "ldx": 1 << 31, "ldq": 1 << 31}, "out of range"), ({"x": None}, "null"),
    ({"q": None}, "null"), ({"scale": None}, "null"), ({"ldx": 7}, "stride"), ({"ldq": 7}, "stride"),
    ({"transpose": 1, "ldq": 2}, "stride"), ({"x": P + 1}, "aligned"), ({"scale": P + 1}, "scales must be aligned")])
def test_quantize_arguments(change, match):
    a = dict(dtype=BF16, x=P, ldx=8, rows=3, cols=8, transpose=0, tile=0, qdtype=E4M3, q=P, ldq=8, sdtype=F32, scale=P, srow=1,
             sblock=3, stream=None)
    a.update(change)
    _refused(_native.load().hcg_quantize_fp8(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"algo": 99}, "unknown algo 99"), ({"algo": -1}, "unknown algo -1"), ({"algo": 256 * 17 + 3}, "unknown algo"),
    ({"algo": 256 * 2}, "unknown algo 512"), ({"xdtype": F16}, "x's type 0"), ({"sdtype": F16}, "scales of type 0"),
    ({"ydtype": E4M3}, "output's type 3"), ({"tokens": -1}, "out of range"), ({"tokens": 1 << 26}, "out of range"),
    ({"outputs": 1 << 26}, "out of range"), ({"inputs": 4000000}, "out of range"), ({"inputs": 0}, "no inputs"),
    ({"x": None}, "null"), ({"w": None}, "null"), ({"xs": None}, "null"), ({"ws": None}, "null"), ({"y": None}, "null"),
    ({"ldx": 7}, "stride"), ({"ldw": 7}, "stride"), ({"ldy": 4}, "stride"), ({"ldx": 4000000}, "strides of 4000000"),
    ({"ldw": 4000000}, "strides of"), ({"y": P + 1}, "aligned"), ({"xs": P + 2}, "scales must be aligned"),
    ({"ws": P + 2}, "scales must be aligned")])
def test_linear_arguments(change, match):
    a = dict(algo=0, xdtype=E4M3, x=P, ldx=8, tokens=3, w=P, ldw=8, outputs=5, inputs=8, sdtype=F32, xs=P, xsr=1, xsb=3,
             tile=1, ws=P, wsr=1, wsb=1, ydtype=BF16, y=P, ldy=5, work=P, bytes=1 << 30, stream=None)
    a.update(change)
    _refused(_native.load().hcg_linear_fp8(*a.values()), match)


def test_calls_without_work_launch_nothing():
    lib = _native.load()
    assert lib.hcg_rms_norm(BF16, None, 8, 0, 8, BF16, None, 0, BF16, None, 1e-6, None, 8, None, 8, None, None) == 0
    assert lib.hcg_rms_norm_fp8(BF16, None, 8, 0, 8, BF16, None, 0, BF16, None, 1e-6, E4M3, None, 8, F32, None, 1, 1, None, 8,
                                None, None) == 0
    assert lib.hcg_quantize_fp8(BF16, None, 8, 0, 8, 0, 0, E4M3, None, 8, F32, None, 1, 1, None) == 0
    assert lib.hcg_linear_fp8(0, E4M3, None, 8, 0, None, 8, 5, 8, F32, None, 1, 1, 1, None, 1, 1, BF16, None, 5, None, 0,
                              None) == 0
    assert lib.hcg_rms_norm_grad_workspace(0, 64) == 0


def test_tensors_must_live_on_a_gpu():
    x, s = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((4, 1))
    q = torch.zeros((4, 8), dtype=torch.float8_e4m3fn)
    for call in (lambda: g.rms_norm(x), lambda: g.rms_norm_grad(x, x, s[:, 0]), lambda: g.rms_norm_fp8(x),
                 lambda: g.quantize_fp8(x), lambda: g.linear_fp8(q, s, q, s)):
        with pytest.raises(LaunchError, match="GPU"):
            call()
    with pytest.raises(LaunchError, match="torch tensor"):
        g.quantize_fp8([1.0, 2.0])
    with pytest.raises(LaunchError, match="torch tensor"):
        g.linear_fp8([1.0], s, q, s)
