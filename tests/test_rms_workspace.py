"""The scratch of the root-mean-square norm's gradient: as many rows of sums as
there are, on the host, and no byte more written, on the GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc.gfx950 import _native  # noqa: E402

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
CODES = {F16: _native.HCG_F16, BF16: _native.HCG_BF16, F32: _native.HCG_F32}


@pytest.mark.parametrize("rows,width,parts", [
    (1, 8, 1), (1, 16384, 1), (1, 1 << 20, 1), (1, 1 << 30, 1), (3, 4096, 3), (255, 4096, 255), (256, 4096, 256),
    (100000, 4096, 256), (100000, 16384, 256), (63, 16385, 63), (64, 16385, 64), (100000, 16385, 64), (70, 1 << 24, 64)])
def test_rows_of_sums(rows, width, parts):
    assert _native.load().hcg_rms_norm_grad_workspace(rows, width) == parts * width * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wide", [(F16, F16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("rows,width", [(1, 3), (300, 3), (33, 100), (9000, 100), (1, 4096), (300, 4096), (700, 9000),
                                        (300, 16384), (70, 16385), (1, 1 << 20)])
def test_no_more_is_written(rows, width, dtype, wide):
    gen = torch.Generator(device=DEV).manual_seed(rows + width)
    dy = torch.randn((rows, width), generator=gen, device=DEV).to(dtype)
    h = torch.randn((rows, width), generator=gen, device=DEV).to(wide)
    rstd = torch.rand((rows,), generator=gen, device=DEV) + 0.5
    want_dh, want_dw = g.rms_norm_grad(dy, h, rstd)
    lib = _native.lib()
    need = lib.hcg_rms_norm_grad_workspace(rows, width)
    buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    dh, dw = torch.empty_like(h), torch.empty((width,), dtype=dtype, device=DEV)
    rc = lib.hcg_rms_norm_grad(CODES[dtype], dy.data_ptr(), width, CODES[wide], h.data_ptr(), width, rows, width,
                               rstd.data_ptr(), CODES[dtype], None, None, 0, dh.data_ptr(), width, dw.data_ptr(),
                               buf.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(dh, want_dh) and torch.equal(dw, want_dw)
    assert (buf[need:] == 0xA5).all()
