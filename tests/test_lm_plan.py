"""hcg_linear_cross_entropy_plan, and that the sizes of the head's GPU tests
reach every tile shape of its three products."""

from __future__ import annotations

import ctypes

import pytest

pytest.importorskip("torch")

from hc.gfx950 import _native

from .test_lm_gpu import _HEADS
from .test_lm_head_gpu import HEADS


def _plan(tokens, vocab, width, grad):
    plan = (ctypes.c_int * 10)()
    rc = _native.load().hcg_linear_cross_entropy_plan(tokens, vocab, width, grad, plan)
    assert rc == 0, _native.last_error(_native.load())
    return plan[0], [tuple(plan[i : i + 3]) for i in (1, 4, 7)]


def test_plan():
    pieces, (logits, dx, dw) = _plan(8192, 32768, 2048, 1)
    assert pieces == 1 and logits == dx == dw == (256, 256, 1)
    assert _plan(8192, 32768, 2048, 0) == (1, [(256, 256, 1), (0, 0, 0), (0, 0, 0)])
    assert _plan(9000, 131072, 64, 1)[0] == 3  # 2^29 probabilities in a piece
    lib = _native.load()
    plan = (ctypes.c_int * 10)()
    for sizes in ((0, 5, 5), (1 << 26, 5, 5), (5, 0, 5), (5, 4000000, 5), (5, 5, 0), (5, 5, 4000000)):
        assert lib.hcg_linear_cross_entropy_plan(*sizes, 1, plan) == _native.HCG_EINVAL
    assert lib.hcg_linear_cross_entropy_plan(5, 5, 5, 1, None) == _native.HCG_EINVAL


def test_the_gpu_tests_reach_every_shape():
    seen = {"loss": set(), "logits": set(), "dx": set(), "dw": set()}
    several = set()
    for size in _HEADS + HEADS:
        pieces, products = _plan(*size, 1)
        for name, (m, n, parts) in zip(("logits", "dx", "dw"), products):
            seen[name].add((m, n, parts > 1))
            if pieces > 1:
                several.add((name, m, n))
        m, n, parts = _plan(*size, 0)[1][0]
        seen["loss"].add((m, n, parts > 1))
    shapes = [(256, 256), (128, 128), (128, 64), (128, 32)]
    whole = {(m, n, False) for m, n in shapes}
    # Small tiles split in every product, the others in dx.
    assert seen["loss"] == seen["logits"] == whole | {(128, 64, True), (128, 32, True)}
    assert seen["dx"] == whole | {(m, n, True) for m, n in shapes}
    assert seen["dw"] == whole - {(128, 32, False)} | {(128, 64, True)}
    assert several == {(name, 256, 256) for name in ("logits", "dx", "dw")}
