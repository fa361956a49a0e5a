"""The language-model operators without a GPU: the library exports what
include/hcg_lm.h declares, bad arguments are rejected on the host before any
launch, and the Python entry points refuse tensors that are not on a GPU."""

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
P = 0x1000  # any non-null, aligned pointer: a rejected call never reads it


def test_header_and_library_agree():
    text = open(os.path.join(ROOT, "include", "hcg_lm.h")).read()
    declared = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(hcg_\w+)\s*\(", text, re.M)))
    assert declared == sorted(_native.LM_EXPORTS)
    lib = _native.load()
    for name in declared:
        assert hasattr(lib, name), name
    assert re.search(r"#define HCG_F32 (\d+)", text).group(1) == str(F32)


def _refused(rc, match):
    assert rc == _native.HCG_EINVAL
    assert re.search(match, _native.last_error(_native.load())), _native.last_error(_native.load())


@pytest.mark.parametrize("change,match", [
    ({"dtype": 3}, "dtype 3"), ({"id_bytes": 2}, "4 or 8 bytes"), ({"n": -1}, "out of range"),
    ({"n": 1 << 30}, "out of range"), ({"width": 1 << 30}, "out of range"), ({"vocab": -2}, "out of range"),
    ({"table": None}, "null"), ({"ids": None}, "null"), ({"out": None}, "null"), ({"ldt": 7}, "stride"),
    ({"ldo": 7}, "stride"), ({"table": P + 1}, "aligned"), ({"ids": P + 4}, "aligned")])
def test_embedding_arguments(change, match):
    a = dict(dtype=BF16, table=P, ldt=8, vocab=5, width=8, id_bytes=8, ids=P, n=3, scale=1.0, out=P, ldo=8, stream=None)
    a.update(change)
    _refused(_native.load().hcg_embedding(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"dtype": -1}, "dtype -1"), ({"grad_dtype": F16}, "type of dy or float32"), ({"id_bytes": 1}, "4 or 8 bytes"),
    ({"vocab": 1 << 30}, "out of range"), ({"n": -3}, "out of range"), ({"width": 1 << 23}, "out of range"),
    ({"dy": None}, "null"), ({"grad": None}, "null"), ({"lddy": 7}, "stride"), ({"ldg": 7}, "stride"),
    ({"grad": P + 2, "grad_dtype": F32}, "aligned"), ({"ws": None}, "workspace"), ({"ws_bytes": 100}, "workspace of 100"),
    ({"ws": P + 8}, "workspace")])
def test_embedding_grad_arguments(change, match):
    lib = _native.load()
    a = dict(dtype=BF16, dy=P, lddy=8, n=5000, width=8, id_bytes=8, ids=P, vocab=5, padding=-1, scale=1.0,
             grad_dtype=BF16, grad=P, ldg=8, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(change)
    _refused(lib.hcg_embedding_grad(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"dtype": 9}, "dtype 9"), ({"pdtype": F16}, "type or float32"), ({"rows": -1}, "out of range"),
    ({"rows": 1 << 31}, "out of range"), ({"width": (1 << 30) + 1}, "out of range"), ({"width": 0}, "without elements"),
    ({"x": None}, "null"), ({"y": None}, "null"), ({"ldx": 7}, "stride"), ({"ldy": 7}, "stride"), ({"x": P + 1}, "aligned")])
def test_layer_norm_arguments(change, match):
    a = dict(dtype=BF16, x=P, ldx=8, rows=3, width=8, pdtype=BF16, weight=P, bias=P, eps=1e-5, y=P, ldy=8, mean=P,
             rstd=P, stream=None)
    a.update(change)
    _refused(_native.load().hcg_layer_norm(*a.values()), match)


@pytest.mark.parametrize("change,match", [
    ({"dtype": 9}, "dtype 9"), ({"pdtype": F16}, "type or float32"), ({"rows": 1 << 31}, "out of range"),
    ({"width": 0}, "without elements"), ({"dy": None}, "null"), ({"mean": None}, "null"), ({"dx": None}, "null"),
    ({"lddy": 7}, "stride"), ({"lddx": 7}, "stride"), ({"dx": P + 1}, "aligned"), ({"ws": None}, "workspace"),
    ({"ws_bytes": 8}, "workspace of 8")])
def test_layer_norm_grad_arguments(change, match):
    a = dict(dtype=BF16, dy=P, lddy=8, x=P, ldx=8, rows=3, width=8, mean=P, rstd=P, pdtype=BF16, weight=P, dx=P,
             lddx=8, dw=P, db=P, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(change)
    _refused(_native.load().hcg_layer_norm_grad(*a.values()), match)


_HEAD = [({"dtype": F32}, "not HCG_F16 or HCG_BF16"), ({"id_bytes": 3}, "4 or 8 bytes"), ({"tokens": -1}, "out of range"),
         ({"tokens": 1 << 26}, "out of range"), ({"vocab": 4000000}, "out of range"), ({"width": 4000000}, "out of range"),
         ({"vocab": 0}, "no vocabulary"), ({"width": 0}, "without elements"), ({"x": None}, "null"),
         ({"weight": None}, "null"), ({"targets": None}, "null"), ({"loss": None}, "null"), ({"ldx": 7}, "stride"),
         ({"ldw": 7}, "stride"), ({"x": P + 1}, "aligned"), ({"targets": P + 4}, "aligned"), ({"ws": None}, "workspace"),
         ({"ws_bytes": 256}, "workspace of 256"), ({"ws": P + 16}, "256-byte aligned")]


@pytest.mark.parametrize("change,match", _HEAD + [({"lse": None}, "null")])
def test_linear_cross_entropy_arguments(change, match):
    a = dict(dtype=BF16, x=P, ldx=8, tokens=3, weight=P, ldw=8, vocab=5, width=8, id_bytes=8, targets=P, ignore=-100,
             loss=P, lse=P, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(change)
    _refused(_native.load().hcg_linear_cross_entropy(*a.values()), match)


@pytest.mark.parametrize("change,match", _HEAD + [({"dx": None}, "null"), ({"dw": None}, "null"), ({"lddx": 7}, "stride"),
                                                  ({"lddw": 7}, "stride"), ({"dw": P + 1}, "aligned")])
def test_linear_cross_entropy_grad_arguments(change, match):
    a = dict(dtype=F16, x=P, ldx=8, tokens=3, weight=P, ldw=8, vocab=5, width=8, id_bytes=8, targets=P, ignore=-100,
             mean=1, scale=1.0, loss=P, dx=P, lddx=8, dw=P, lddw=8, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(change)
    _refused(_native.load().hcg_linear_cross_entropy_grad(*a.values()), match)


def test_workspace_sizes():
    lib = _native.load()
    assert lib.hcg_embedding_grad_workspace(BF16, 16, 1000, 1 << 20) == 0  # too few tokens for a long row
    assert lib.hcg_embedding_grad_workspace(BF16, 17, 1000, 1 << 20) > 0
    assert lib.hcg_embedding_grad_workspace(BF16, 2048, 1000, 2048) == 0  # one launch
    assert lib.hcg_embedding_grad_workspace(F32, 2048, 1000, 2048) > 0
    assert lib.hcg_embedding_grad_workspace(BF16, 4096, 1000, 1024) == 0
    assert lib.hcg_embedding_grad_workspace(BF16, 2049, 1000, 1032) > 0
    assert lib.hcg_embedding_grad_workspace(BF16, 4097, 1000, 64) > 0
    assert lib.hcg_embedding_grad_workspace(BF16, 0, 0, 0) == 0
    assert lib.hcg_layer_norm_grad_workspace(0, 64) == 0
    size = lib.hcg_linear_cross_entropy_workspace
    assert size(0, 100, 64, P, 64, 1) == 0
    # the logits' gradient is held for at most 1 GiB of tokens
    small, large = size(4096, 131072, 64, P, 64, 1), size(65536, 131072, 64, P, 64, 1)
    assert (1 << 30) <= small < (1 << 30) * 1.2 and large < (1 << 30) * 1.2
    # forward only: nothing of tokens x vocabulary
    assert size(65536, 131072, 64, P, 64, 0) < 65536 * 131072 // 8
    # a weight whose rows are not 16-byte aligned is copied
    assert size(64, 5000, 64, P + 2, 64, 0) - size(64, 5000, 64, P, 64, 0) == 5000 * 64 * 2


def test_calls_without_work_launch_nothing():
    lib = _native.load()
    assert lib.hcg_embedding(BF16, None, 8, 0, 8, 8, None, 0, 1.0, None, 8, None) == 0
    assert lib.hcg_embedding_grad(BF16, None, 8, 0, 8, 8, None, 0, -1, 1.0, BF16, None, 8, None, 0, None) == 0
    assert lib.hcg_layer_norm(BF16, None, 8, 0, 8, BF16, None, None, 1e-5, None, 8, None, None, None) == 0
    assert lib.hcg_linear_cross_entropy(BF16, None, 8, 0, None, 8, 5, 8, 8, None, -100, None, None, None, 0, None) == 0


def test_tensors_must_live_on_a_gpu():
    x, ids = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    s = torch.zeros(4)
    for call in (lambda: g.embedding(ids, x), lambda: g.embedding_grad(x, ids, 5), lambda: g.layer_norm(x),
                 lambda: g.layer_norm_grad(x, x, s, s), lambda: g.linear_cross_entropy(x, x, ids),
                 lambda: g.linear_cross_entropy_grad(x, x, ids)):
        with pytest.raises(LaunchError, match="GPU"):
            call()
    with pytest.raises(LaunchError, match="torch tensor"):
        g.layer_norm([1.0, 2.0])
