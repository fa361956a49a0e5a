"""Linear layers in 8-bit floating point on gfx950.

A quantised matrix is a pair ``(q, scale)``: ``q`` (rows x cols) of
``torch.float8_e4m3fn`` or ``torch.float8_e5m2`` and a scale for each 128
columns of each row, ``scale`` being (rows x ceil(cols / 128)), or of each 128 x
128 tile, (ceil(rows / 128) x ceil(cols / 128)).  Element (r, c) stands for
``q[r, c] * scale[r or r // 128, c // 128]``.  Scales are float32, or
``torch.float8_e8m0fnu``, powers of two, which the matrix instructions take as
they are.

    q, s, h, rstd = rms_norm_fp8(x, weight, residual)   # activations
    qw, sw = quantize_fp8(w, block="tile")              # a layer's weight, (outputs x inputs)
    y = linear_fp8(q, s, qw, sw)

and its gradients, from dy (tokens x outputs):

    dx = linear_fp8(*quantize_fp8(dy, dtype=torch.float8_e5m2), *quantize_fp8(w, block="tile", transpose=True))
    dw = linear_fp8(*quantize_fp8(dy, transpose=True, dtype=torch.float8_e5m2),
                    *quantize_fp8(x, transpose=True), out_dtype=torch.float32)

The entry points take torch tensors on a GPU and run in libhcg_gfx950.so
(include/hcg_fp8.h) as those of :mod:`hc.gfx950.lm` do: on the tensors' device
and current stream, asynchronously, with arguments checked before anything is
launched (``LaunchError``).  Results are the same from run to run, and carry no
autograd graph.
"""

from __future__ import annotations

import math
from typing import Any

from .._errors import LaunchError
from . import _native, lm
from .lm import (_ANY, _CODES, _call, _check_tensor, _code, _fast, _finish, _ld, _name, _out_rows, _ptr, _rms_args,
                 _rows)

_Q_CODES: dict[Any, int] = {}      # torch dtype -> HCG_E4M3, HCG_E5M2
_SCALE_CODES: dict[Any, int] = {}  # torch dtype -> HCG_F32, HCG_E8M0


def _torch() -> Any:
    torch = lm._torch()
    if not _Q_CODES:
        _SCALE_CODES.update({torch.float32: _native.HCG_F32, torch.float8_e8m0fnu: _native.HCG_E8M0})
        _Q_CODES.update({torch.float8_e4m3fn: _native.HCG_E4M3, torch.float8_e5m2: _native.HCG_E5M2})
    return torch


def _blocks(n: int) -> int:
    return -(-n // _native.FP8_BLOCK)


def _types(torch: Any, dtype: Any, scale_dtype: Any) -> tuple[Any, Any]:
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    scale_dtype = torch.float32 if scale_dtype is None else scale_dtype
    if dtype not in _Q_CODES:
        raise LaunchError(f"dtype must be float8_e4m3fn or float8_e5m2, got {_name(dtype)}")
    if scale_dtype not in _SCALE_CODES:
        raise LaunchError(f"scale_dtype must be float32 or float8_e8m0fnu, got {_name(scale_dtype)}")
    return dtype, scale_dtype


def _new(torch: Any, lead: tuple[int, ...], last: int, first: int, step: int, dtype: Any, device: Any) -> Any:
    """A tensor of shape lead + (last,): rows `first` apart, their elements `step`."""
    strides = [step]
    for n in reversed(lead):
        strides.insert(0, first)
        first *= max(n, 1)
    return torch.empty_strided((*lead, last), strides, dtype=dtype, device=device)


def _new_q(torch: Any, lead: tuple[int, ...], cols: int, dtype: Any, device: Any) -> tuple[Any, int]:
    """(q of shape lead + (cols,), its row stride): rows start at multiples of
    16 bytes, as the product reads them in place."""
    ld = max(-(-cols // 16) * 16, 1)
    return _new(torch, lead, cols, ld, 1, dtype, device), ld


def _new_scale(torch: Any, lead: tuple[int, ...], blocks: int, dtype: Any, device: Any) -> tuple[Any, int]:
    """(scale of shape lead + (blocks,), the stride between its blocks): block
    by block in memory, so that neighbouring rows' lie next to each other."""
    step = max(math.prod(lead), 1)
    return _new(torch, lead, blocks, 1, step, dtype, device), step


def quantize_fp8(x: Any, *, block: str = "row", transpose: bool = False, dtype: Any | None = None,
                 scale_dtype: Any | None = None) -> tuple[Any, Any]:
    """``(q, scale)`` of ``x`` (float16, bfloat16 or float32; leading
    dimensions are rows), or with ``transpose`` of its transpose, (cols x rows)
    whatever x's leading dimensions.

    ``block``: ``"row"``, a scale for each 128 columns of each row of q, or
    ``"tile"``, for each 128 x 128 of them.  With a = max(largest magnitude of
    the block, 2^-100) and F the largest value of ``dtype`` (float8_e4m3fn, the
    default: 448; float8_e5m2: 57344), a float32 scale is a / F and q is x * (F /
    a), rounded to nearest; a float8_e8m0fnu scale is the least power of two not
    below a / F.  A block that holds an infinity or a NaN stands for NaN."""
    torch = _torch()
    if block not in ("row", "tile"):
        raise LaunchError(f"unknown block {block!r}; expected 'row' or 'tile'")
    dtype, scale_dtype = _types(torch, dtype, scale_dtype)
    r = _fast("quantize_fp8", x, block == "tile", bool(transpose), _Q_CODES[dtype], _SCALE_CODES[scale_dtype])
    if r is not None:
        return r
    index = _check_tensor(torch, x, "x")
    code = _code(x, "x", _ANY)
    rows = _rows(x, "x")
    n, cols = rows.shape
    lead, across = ((cols,), n) if transpose else (tuple(x.shape[:-1]), cols)
    q, ldq = _new_q(torch, lead, across, dtype, x.device)
    down = (_blocks(cols if transpose else n),) if block == "tile" else lead
    scale, step = _new_scale(torch, down, _blocks(across), scale_dtype, x.device)
    _call(torch, index, _native.lib().hcg_quantize_fp8, "hcg_quantize_fp8", code, _ptr(rows), _ld(rows), n, cols,
          bool(transpose), block == "tile", _Q_CODES[dtype], _ptr(q), ldq, _SCALE_CODES[scale_dtype], _ptr(scale), 1,
          step)
    return q, scale


def rms_norm_fp8(x: Any, weight: Any | None = None, residual: Any | None = None, *, eps: float = 1e-6,
                 dtype: Any | None = None, scale_dtype: Any | None = None) -> tuple[Any, Any, Any, Any]:
    """:func:`hc.gfx950.rms_norm` with the result quantised by rows, as
    :func:`quantize_fp8` does, before any other rounding: ``(q, scale, h,
    rstd)``, where q and scale stand for ``h * rstd * weight``."""
    torch = _torch()
    dtype, scale_dtype = _types(torch, dtype, scale_dtype)
    r = _fast("rms_norm_fp8", x, weight, residual, eps, _Q_CODES[dtype], _SCALE_CODES[scale_dtype])
    if r is not None:
        return r if residual is not None else (r[0], r[1], x, r[3])
    index, code, rows, w, wcode, res, rcode, h, hrows, rstd = _rms_args(torch, x, weight, residual)
    n, width = rows.shape
    lead = tuple(x.shape[:-1])
    q, ldq = _new_q(torch, lead, width, dtype, x.device)
    scale, step = _new_scale(torch, lead, _blocks(width), scale_dtype, x.device)
    _call(torch, index, _native.lib().hcg_rms_norm_fp8, "hcg_rms_norm_fp8", code, _ptr(rows), _ld(rows), n, width, rcode,
          _ptr(res), 0 if res is None else _ld(res), wcode, _ptr(w), eps, _Q_CODES[dtype], _ptr(q), ldq,
          _SCALE_CODES[scale_dtype], _ptr(scale), 1, step, _ptr(hrows), width, _ptr(rstd))
    return q, scale, h, rstd


def _scale_arg(torch: Any, scale: Any, what: str, index: int) -> int:
    _check_tensor(torch, scale, what, index)
    code = _SCALE_CODES.get(scale.dtype)
    if code is None:
        raise LaunchError(f"{what} must be float32 or float8_e8m0fnu, got {_name(scale.dtype)}")
    return code


def _algo_number(algo: Any) -> int:
    """HCG_FP8_* of a form's name, or of "128x128/4", K in four parts."""
    name, _, splits = str(algo).partition("/")
    number = _native.FP8_ALGOS.get(name)
    plain = splits.isascii() and splits.isdigit() and len(splits) < 9
    parts = int(splits) if plain else 0
    if number is None or (splits and not plain) or parts > _native.FP8_MAX_SPLITS or (number == 0 and parts):
        raise LaunchError(f"unknown algo {algo!r}; expected one of {', '.join(_native.FP8_ALGOS)}, the forms after auto "
                          f"also with /1 to /{_native.FP8_MAX_SPLITS} for so many parts of the inputs")
    return number + _native.FP8_SPLITS * parts


def linear_fp8(x: Any, x_scale: Any, weight: Any, weight_scale: Any, *, out_dtype: Any | None = None,
               out: Any | None = None, algo: str = "auto") -> Any:
    """``x @ weight.T`` of two quantised matrices: ``x`` (..., inputs),
    float8_e4m3fn or float8_e5m2, with ``x_scale`` (..., ceil(inputs / 128)), and
    ``weight`` (outputs x inputs), float8_e4m3fn, with a scale for each row
    (outputs x ceil(inputs / 128)) or each tile (ceil(outputs / 128) x ...); both
    scales float32 or both float8_e8m0fnu, in any strides.

    The result is (..., outputs) of ``out_dtype`` (bfloat16, the default, float16
    or float32; that of ``out``).  A float32 one has float32 sums of exact
    products, at the rate of 16-bit products.  A 16-bit one comes from the 8-bit
    matrix instructions: sums are float32, but each product is cut below 2^-13 of
    the largest among 8 neighbours (1.5e-5 of the results for normal operands, up
    to 8e-5 where a few columns are much larger than the others) before the result's
    own rounding.  ``algo`` forces a form, for measurements.  Rows that start at multiples of 16 bytes, as
    :func:`quantize_fp8` makes them, are read where they lie."""
    torch = _torch()
    if out is None and algo == "auto":
        code = _CODES.get(torch.bfloat16 if out_dtype is None else out_dtype)
        if code is not None:
            r = _fast("linear_fp8", x, x_scale, weight, weight_scale, code)
            if r is not None:
                return r
    index = _check_tensor(torch, x, "x")
    if x.dtype not in _Q_CODES:
        raise LaunchError(f"x must be float8_e4m3fn or float8_e5m2, got {_name(x.dtype)}")
    _check_tensor(torch, weight, "weight", index)
    if weight.dtype is not torch.float8_e4m3fn:
        raise LaunchError(f"weight must be float8_e4m3fn, got {_name(weight.dtype)}")
    if weight.ndim != 2 or x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise LaunchError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} (outputs x inputs) do not match")
    code = _scale_arg(torch, x_scale, "x_scale", index)
    if _scale_arg(torch, weight_scale, "weight_scale", index) != code:
        raise LaunchError(f"x_scale and weight_scale must have one type, got {_name(x_scale.dtype)} and "
                          f"{_name(weight_scale.dtype)}")
    outputs, inputs = weight.shape
    blocks = _blocks(inputs)
    if tuple(x_scale.shape) != (*x.shape[:-1], blocks):
        raise LaunchError(f"x_scale shape {tuple(x_scale.shape)} does not match {(*x.shape[:-1], blocks)}")
    tile = tuple(weight_scale.shape) == (_blocks(outputs), blocks)
    if not tile and tuple(weight_scale.shape) != (outputs, blocks):
        raise LaunchError(f"weight_scale shape {tuple(weight_scale.shape)} is neither {(outputs, blocks)} (rows) nor "
                          f"{(_blocks(outputs), blocks)} (tiles)")
    number = _algo_number(algo)
    if out is not None:
        out_dtype = out.dtype if out_dtype is None and isinstance(out, torch.Tensor) else out_dtype
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    if out_dtype not in _CODES:
        raise LaunchError(f"the output must be float16, bfloat16 or float32, got {_name(out_dtype)}")
    rows, w = _rows(x, "x"), _rows(weight, "weight")
    tokens = rows.shape[0]
    if inputs == 0 and tokens and outputs:
        raise LaunchError("a product over no inputs")
    xs = x_scale.reshape(tokens, blocks)
    shape = (*x.shape[:-1], outputs)
    if out is None:
        out = m = torch.empty(shape, dtype=out_dtype, device=x.device)
        ldo = max(outputs, 1)
    else:
        out, m = _out_rows(torch, out, shape, out_dtype, "out", index)
        ldo = _ld(m)
    lib = _native.lib()
    need = lib.hcg_linear_fp8_workspace(number, tokens, outputs, inputs, _ptr(rows), _ld(rows), _ptr(w), _ld(w), code,
                                        xs.stride(0), tile, _ptr(weight_scale), *weight_scale.stride(), _CODES[out_dtype])
    ws = lm._workspace(torch, need, x.device)
    _call(torch, index, lib.hcg_linear_fp8, "hcg_linear_fp8", number, _Q_CODES[x.dtype], _ptr(rows), _ld(rows), tokens,
          _ptr(w), _ld(w), outputs, inputs, code, _ptr(xs), xs.stride(0), xs.stride(1), tile, _ptr(weight_scale),
          weight_scale.stride(0), weight_scale.stride(1), _CODES[out_dtype], _ptr(m), ldo, _ptr(ws), need)
    return out if m is out else _finish(out, m)
