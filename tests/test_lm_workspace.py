"""The scratch of layer norm's gradient: as many rows of sums as there are, on
the host, and no byte more written, on the GPU."""

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
    assert _native.load().hcg_layer_norm_grad_workspace(rows, width) == parts * 2 * width * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,width", [(1, 3), (300, 3), (33, 100), (9000, 100), (1, 4096), (300, 4096), (700, 9000),
                                        (300, 16384), (70, 16385), (1, 1 << 20)])
def test_no_more_is_written(rows, width, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows + width)
    dy, x = (torch.randn((rows, width), generator=gen, device=DEV).to(dtype) for _ in range(2))
    mean = torch.rand((rows,), generator=gen, device=DEV) - 0.5
    rstd = torch.rand((rows,), generator=gen, device=DEV) + 0.5
    want = g.layer_norm_grad(dy, x, mean, rstd)
    lib = _native.lib()
    need = lib.hcg_layer_norm_grad_workspace(rows, width)
    buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    dx, dw, db = torch.empty_like(x), torch.empty((width,), dtype=dtype, device=DEV), torch.empty((width,), dtype=dtype,
                                                                                                  device=DEV)
    rc = lib.hcg_layer_norm_grad(CODES[dtype], dy.data_ptr(), width, x.data_ptr(), width, rows, width, mean.data_ptr(),
                                 rstd.data_ptr(), CODES[dtype], None, dx.data_ptr(), width, dw.data_ptr(), db.data_ptr(),
                                 buf.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    for got, w in zip((dx, dw, db), want):
        assert torch.equal(got, w)
    assert (buf[need:] == 0xA5).all()
