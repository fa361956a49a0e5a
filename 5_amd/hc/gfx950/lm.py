"""The two ends of a language model on gfx950, and the norm between them.

``embedding``, ``layer_norm`` and ``linear_cross_entropy`` with their
gradients, for training beside the products of :func:`hc.gfx950.gemm`.  They
take torch tensors on a GPU and run in libhcg_gfx950.so (include/hcg_lm.h) on
the tensors' device and current stream, asynchronously; arguments are checked
before anything is launched and raise ``LaunchError``.  Leading dimensions are
rows: an activation is ``(..., width)``.  Rows may be strided views; other
layouts are copied.  Sums and statistics are float32, a 16-bit result is
rounded once (the head's gradient holds two intermediates in 16 bits, see
there), and every result is the same from run to run.

The gradients are calls of their own: outputs carry no autograd graph, also
where inputs require gradients.
"""

from __future__ import annotations

import sys
from typing import Any

from .._errors import LaunchError
from . import _native

_PKG = sys.modules[__package__]  # hc.gfx950 (still loading here): torch, the current device and stream

_CODES: dict[Any, int] = {}  # torch dtype -> HCG_*
_ID_BYTES: dict[Any, int] = {}


def _torch() -> Any:
    torch = _PKG._torch()
    if not _CODES:
        _ID_BYTES.update({torch.int32: 4, torch.int64: 8})
        _CODES.update({torch.float16: _native.HCG_F16, torch.bfloat16: _native.HCG_BF16,
                       torch.float32: _native.HCG_F32})
    return torch


_FAST: Any = None  # _hcg_torch once loaded; False where it is not built


def _fast(name: str, *args: Any) -> Any:
    """The compiled binding's result for contiguous tensors on the current
    device (a call costs about 10 us less host time than below), or None: the
    general path below takes the call, or says what is wrong with it."""
    global _FAST
    if _FAST is None:
        _FAST = _PKG._fast_gemm() and sys.modules[__package__ + "._hcg_torch"]
    if not _FAST:
        return None
    try:
        result = getattr(_FAST, name)(*args)
    except TypeError:  # an argument that is no tensor or number
        return None
    if type(result) is int:
        _native.check(_native.lib(), result, "hcg_" + name)
    return result


def _name(dtype: Any) -> str:
    return str(dtype).replace("torch.", "")


def _check_tensor(torch: Any, t: Any, what: str, index: int | None = None) -> int:
    """The tensor's device index, which is ``index`` where that is given."""
    if not isinstance(t, torch.Tensor):
        raise LaunchError(f"{what} must be a torch tensor, got {type(t).__name__}")
    d = t.get_device()
    if d < 0:
        raise LaunchError(f"{what} must live on a GPU")
    if index is not None and d != index:
        raise LaunchError(f"{what} must live on the same device as the other tensors")
    return d


def _code(t: Any, what: str, allowed: tuple[int, ...]) -> int:
    code = _CODES.get(t.dtype)
    if code is None or code not in allowed:
        names = " or ".join(_name(d) for d, c in _CODES.items() if c in allowed)
        raise LaunchError(f"{what} must be {names}, got {_name(t.dtype)}")
    return code


_ANY = (_native.HCG_F16, _native.HCG_BF16, _native.HCG_F32)
_HALF = (_native.HCG_F16, _native.HCG_BF16)


def _rows(t: Any, what: str) -> Any:
    """``t`` as a matrix of its last dimension's rows, elements of a row
    next to each other: a view where the strides allow it, else a copy."""
    if t.ndim == 0:
        raise LaunchError(f"{what} must have at least one dimension")
    m = t if t.ndim == 2 else t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((0, t.shape[-1]))
    rows, width = m.shape
    if (width > 1 and m.stride(1) != 1) or (rows > 1 and m.stride(0) < width):
        m = m.contiguous()
    return m


def _ld(m: Any) -> int:
    return m.stride(0) if m.shape[0] > 1 else max(m.shape[1], 1)


def _out_rows(torch: Any, out: Any, shape: tuple[int, ...], dtype: Any, what: str, index: int) -> tuple[Any, Any]:
    """(out, the matrix to write): the matrix is a view of ``out`` where its
    strides allow it, else scratch that the caller copies to ``out``."""
    _check_tensor(torch, out, what, index)
    if tuple(out.shape) != shape:
        raise LaunchError(f"{what} shape {tuple(out.shape)} does not match {shape}")
    if out.dtype != dtype:
        raise LaunchError(f"{what} must be {_name(dtype)}, got {_name(out.dtype)}")
    rows = out.numel() // shape[-1] if shape[-1] else 0
    try:
        m = out.view(rows, shape[-1])
    except RuntimeError:
        return out, torch.empty((rows, shape[-1]), dtype=dtype, device=out.device)
    if (shape[-1] > 1 and m.stride(1) != 1) or (rows > 1 and m.stride(0) < shape[-1]):
        return out, torch.empty((rows, shape[-1]), dtype=dtype, device=out.device)
    return out, m


def _finish(out: Any, m: Any) -> Any:
    if m.data_ptr() != out.data_ptr() and out.numel():
        out.copy_(m.view(out.shape))
    return out


def _call(torch: Any, index: int, fn: Any, what: str, *args: Any) -> None:
    """fn(*args, stream), on device ``index``."""
    if _PKG._current_device(torch) == index:
        rc = fn(*args, _PKG._current_stream(torch, index) or None)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _PKG._current_stream(torch, index) or None)
    if rc:
        _native.check(_native.lib(), rc, what)


def _ids(torch: Any, t: Any, what: str, index: int) -> tuple[Any, int]:
    _check_tensor(torch, t, what, index)
    size = _ID_BYTES.get(t.dtype)
    if size is None:
        raise LaunchError(f"{what} must be int32 or int64, got {_name(t.dtype)}")
    return (t if t.is_contiguous() else t.contiguous()), size


def _whole(value: Any, what: str) -> int:
    try:
        n = int(value)
    except (TypeError, ValueError, OverflowError):
        n = None
    if n is None or n != value or not -(1 << 63) <= n < 1 << 63:
        raise LaunchError(f"{what} must be a whole number of 64 bits, got {value!r}")
    return n


def _workspace(torch: Any, size: int, device: Any) -> Any:
    # From torch's allocator, which hands memory freed on a stream to later
    # work on that stream only.
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _ptr(t: Any) -> int | None:
    return None if t is None else t.data_ptr() or None


# --------------------------------------------------------------------------
# Embedding
# --------------------------------------------------------------------------


def embedding(tokens: Any, table: Any, *, scale: float = 1.0, out: Any | None = None) -> Any:
    """``scale * table[tokens]``: the rows of ``table`` (vocabulary x width;
    float16, bfloat16 or float32) that ``tokens`` (int32 or int64, any shape)
    name, of shape ``tokens.shape + (width,)``.  A token outside the
    vocabulary gives a row of NaN."""
    if out is None:
        r = _fast("embedding", tokens, table, scale)
        if r is not None:
            return r
    torch = _torch()
    index = _check_tensor(torch, table, "table")
    code = _code(table, "table", _ANY)
    if table.ndim != 2:
        raise LaunchError(f"table must be 2-D, got {table.ndim}-D")
    ids, size = _ids(torch, tokens, "tokens", index)
    rows = _rows(table, "table")
    vocab, width = rows.shape
    shape = (*tokens.shape, width)
    if out is None:
        out = m = torch.empty(shape, dtype=table.dtype, device=table.device)
        ldo = max(width, 1)
    else:
        out, m = _out_rows(torch, out, shape, table.dtype, "out", index)
        ldo = _ld(m)
    lib = _native.lib()
    _call(torch, index, lib.hcg_embedding, "hcg_embedding", code, _ptr(rows), _ld(rows), vocab, width, size,
          _ptr(ids), ids.numel(), scale, _ptr(m), ldo)
    return out if m is out else _finish(out, m)


def embedding_grad(dy: Any, tokens: Any, vocab: int, *, scale: float = 1.0, padding_idx: int | None = None,
                   dtype: Any | None = None, out: Any | None = None) -> Any:
    """The gradient of :func:`embedding` for its table, (``vocab`` x width):
    row v is ``scale`` times the float32 sum of the rows of ``dy``
    (``tokens.shape + (width,)``) whose token is v, in the order of the
    tokens; zeros where there is none and in row ``padding_idx``.  ``dtype``:
    that of ``dy`` (the default) or float32.  Tokens outside the vocabulary
    reach no row."""
    if padding_idx is None and dtype is None and out is None:
        r = _fast("embedding_grad", dy, tokens, vocab, scale)
        if r is not None:
            return r
    torch = _torch()
    index = _check_tensor(torch, dy, "dy")
    code = _code(dy, "dy", _ANY)
    ids, size = _ids(torch, tokens, "tokens", index)
    if dy.ndim != tokens.ndim + 1 or dy.shape[:-1] != tokens.shape:
        raise LaunchError(f"dy shape {tuple(dy.shape)} does not match tokens {tuple(tokens.shape)}")
    vocab = _whole(vocab, "vocab")
    if vocab < 0:
        raise LaunchError(f"vocab must not be negative, got {vocab}")
    if padding_idx is not None:
        padding_idx = _whole(padding_idx, "padding_idx")
        if not 0 <= padding_idx < vocab:
            raise LaunchError(f"padding_idx {padding_idx} is outside the vocabulary of {vocab}")
    rows = _rows(dy, "dy")
    n, width = rows.shape
    if out is not None:
        dtype = out.dtype if dtype is None and isinstance(out, torch.Tensor) else dtype
    dtype = dy.dtype if dtype is None else dtype
    if dtype is not dy.dtype and dtype is not torch.float32:
        raise LaunchError(f"the gradient must be {_name(dy.dtype)} or float32, got {_name(dtype)}")
    if out is None:
        out = m = torch.empty((vocab, width), dtype=dtype, device=dy.device)
        ldg = max(width, 1)
    else:
        out, m = _out_rows(torch, out, (vocab, width), dtype, "out", index)
        ldg = _ld(m)
    lib = _native.lib()
    need = lib.hcg_embedding_grad_workspace(code, n, vocab, width)
    ws = _workspace(torch, need, dy.device)
    _call(torch, index, lib.hcg_embedding_grad, "hcg_embedding_grad", code, _ptr(rows), _ld(rows), n, width, size,
          _ptr(ids), vocab, -1 if padding_idx is None else padding_idx, scale, _CODES[dtype], _ptr(m), ldg, _ptr(ws),
          need)
    return out if m is out else _finish(out, m)


# --------------------------------------------------------------------------
# Layer norm
# --------------------------------------------------------------------------


def _param(torch: Any, p: Any, what: str, x: Any, index: int, like: Any | None = None) -> Any:
    """A parameter vector of x's width, of x's type or float32 (``like``: and
    of the other parameter's type)."""
    if p is None:
        return None
    _check_tensor(torch, p, what, index)
    if p.ndim != 1 or p.shape[0] != x.shape[-1]:
        raise LaunchError(f"{what} shape {tuple(p.shape)} does not match the width {x.shape[-1]}")
    if p.dtype is not x.dtype and p.dtype is not torch.float32:
        raise LaunchError(f"{what} must be {_name(x.dtype)} or float32, got {_name(p.dtype)}")
    if like is not None and p.dtype is not like.dtype:
        raise LaunchError(f"weight and bias must have one type, got {_name(like.dtype)} and {_name(p.dtype)}")
    return p if p.is_contiguous() else p.contiguous()


def layer_norm(x: Any, weight: Any | None = None, bias: Any | None = None, *, eps: float = 1e-5,
               out: Any | None = None) -> tuple[Any, Any, Any]:
    """Layer norm over the last dimension of ``x`` (float16, bfloat16 or
    float32): ``(y, mean, rstd)`` with ``y = (x - mean) * rstd * weight +
    bias`` of x's type and the rows' mean and ``rstd = 1 / sqrt(var + eps)``
    as float32, which :func:`layer_norm_grad` takes.  ``weight`` and ``bias``:
    vectors of x's type or float32, or None."""
    if out is None:
        r = _fast("layer_norm", x, weight, bias, eps)
        if r is not None:
            return r
    torch = _torch()
    index = _check_tensor(torch, x, "x")
    code = _code(x, "x", _ANY)
    rows = _rows(x, "x")
    n, width = rows.shape
    if width == 0:
        raise LaunchError("layer norm of rows without elements")
    w = _param(torch, weight, "weight", x, index)
    b = _param(torch, bias, "bias", x, index, w)
    params = w if w is not None else b
    device = x.device
    shape = x.shape
    if out is None:
        out = m = torch.empty(shape, dtype=x.dtype, device=device)
        ldo = width
    else:
        out, m = _out_rows(torch, out, tuple(shape), x.dtype, "out", index)
        ldo = _ld(m)
    stats = torch.empty((2, *shape[:-1]), dtype=torch.float32, device=device)
    mean, rstd = stats[0], stats[1]
    lib = _native.lib()
    base = stats.data_ptr()
    _call(torch, index, lib.hcg_layer_norm, "hcg_layer_norm", code, _ptr(rows), _ld(rows), n, width,
          code if params is None else _CODES[params.dtype], _ptr(w), _ptr(b), eps, _ptr(m), ldo, base or None,
          base + 4 * n if base else None)
    return (out if m is out else _finish(out, m)), mean, rstd


def layer_norm_grad(dy: Any, x: Any, mean: Any, rstd: Any, weight: Any | None = None, *,
                    param_dtype: Any | None = None) -> tuple[Any, Any, Any]:
    """The gradients of :func:`layer_norm`, ``(dx, dweight, dbias)``, from
    ``dy`` (x's shape and type) and what the forward call returned.  dweight
    and dbias have the type of ``weight`` (x's without one), or
    ``param_dtype``: x's type or float32.  dx is of ``weight`` as it is,
    whatever ``param_dtype``."""
    if param_dtype is None:
        r = _fast("layer_norm_grad", dy, x, mean, rstd, weight)
        if r is not None:
            return r
    torch = _torch()
    index = _check_tensor(torch, x, "x")
    code = _code(x, "x", _ANY)
    _check_tensor(torch, dy, "dy", index)
    if dy.shape != x.shape:
        raise LaunchError(f"dy shape {tuple(dy.shape)} does not match x {tuple(x.shape)}")
    if dy.dtype is not x.dtype:
        raise LaunchError(f"dy must be {_name(x.dtype)} as x, got {_name(dy.dtype)}")
    rows, grads = _rows(x, "x"), _rows(dy, "dy")
    n, width = rows.shape
    if width == 0:
        raise LaunchError("layer norm of rows without elements")
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        _check_tensor(torch, t, what, index)
        if t.numel() != n or t.dtype is not torch.float32:
            raise LaunchError(f"{what} must be {n} float32 values, got {tuple(t.shape)} {_name(t.dtype)}")
    w = _param(torch, weight, "weight", x, index)
    if param_dtype is None:
        param_dtype = x.dtype if w is None else w.dtype
    elif param_dtype is not x.dtype and param_dtype is not torch.float32:
        raise LaunchError(f"param_dtype must be {_name(x.dtype)} or float32, got {_name(param_dtype)}")
    # The call has one type for the weight and its gradients: the wider of the
    # two, so that the weight is never rounded, and the float32 sums are rounded
    # to param_dtype once, below.
    call_dtype = param_dtype
    if w is not None and w.dtype is not param_dtype:
        call_dtype = torch.float32
        w = w.float()
    device = x.device
    dx = torch.empty(x.shape, dtype=x.dtype, device=device)
    params = torch.empty((2, width), dtype=call_dtype, device=device)
    lib = _native.lib()
    need = lib.hcg_layer_norm_grad_workspace(n, width)
    ws = _workspace(torch, need, device)
    base = params.data_ptr()
    mean, rstd = mean.contiguous(), rstd.contiguous()
    _call(torch, index, lib.hcg_layer_norm_grad, "hcg_layer_norm_grad", code, _ptr(grads), _ld(grads), _ptr(rows),
          _ld(rows), n, width, _ptr(mean), _ptr(rstd), _CODES[call_dtype], _ptr(w), _ptr(dx), width, base,
          base + params.element_size() * width, _ptr(ws), need)
    params = params.to(param_dtype)
    return dx, params[0], params[1]


# --------------------------------------------------------------------------
# Softmax cross entropy of a linear head
# --------------------------------------------------------------------------


def _head_args(torch: Any, x: Any, weight: Any, targets: Any, ignore_index: Any) -> tuple[Any, ...]:
    index = _check_tensor(torch, x, "x")
    code = _code(x, "x", _HALF)
    _check_tensor(torch, weight, "weight", index)
    if weight.dtype is not x.dtype:
        raise LaunchError(f"x and weight must have one type, got {_name(x.dtype)} and {_name(weight.dtype)}")
    if weight.ndim != 2 or x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise LaunchError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} (vocabulary x width) do not match")
    ids, size = _ids(torch, targets, "targets", index)
    if targets.shape != x.shape[:-1]:
        raise LaunchError(f"targets shape {tuple(targets.shape)} does not match x {tuple(x.shape)}")
    if weight.shape[0] == 0 and targets.numel():
        raise LaunchError("a softmax over no vocabulary")
    if weight.shape[1] == 0 and targets.numel():
        raise LaunchError("hidden states without elements")
    return index, code, _rows(x, "x"), _rows(weight, "weight"), ids, size, _whole(ignore_index, "ignore_index")


def linear_cross_entropy(x: Any, weight: Any, targets: Any, *, ignore_index: int = -100) -> tuple[Any, Any]:
    """Per token, the softmax cross entropy of the logits ``x @ weight.T``
    against ``targets``: ``(loss, lse)``, float32 of targets' shape, with
    ``lse = log(sum(exp(logits)))`` and ``loss = lse - logits[target]``.

    x: (..., width), weight: (vocabulary, width), both float16 or both
    bfloat16; targets: int32 or int64.  Tokens whose target is
    ``ignore_index`` have loss and lse 0, whatever x holds there; other
    targets outside the vocabulary give NaN.  The logits are never written."""
    r = _fast("linear_cross_entropy", x, weight, targets, ignore_index)
    if r is not None:
        return r
    torch = _torch()
    index, code, rows, w, ids, size, ignore = _head_args(torch, x, weight, targets, ignore_index)
    n, width = rows.shape
    vocab = w.shape[0]
    out = torch.empty((2, *targets.shape), dtype=torch.float32, device=x.device)
    lib = _native.lib()
    need = lib.hcg_linear_cross_entropy_workspace(n, vocab, width, _ptr(w), _ld(w), 0)
    ws = _workspace(torch, need, x.device)
    if n:
        base = out.data_ptr()
        _call(torch, index, lib.hcg_linear_cross_entropy, "hcg_linear_cross_entropy", code, _ptr(rows), _ld(rows), n,
              _ptr(w), _ld(w), vocab, width, size, _ptr(ids), ignore, base, base + 4 * n, _ptr(ws), need)
    return out[0], out[1]


def linear_cross_entropy_grad(x: Any, weight: Any, targets: Any, *, ignore_index: int = -100,
                              reduction: str = "mean", grad_scale: float = 1.0) -> tuple[Any, Any, Any]:
    """``(loss, dx, dweight)``: the loss of :func:`linear_cross_entropy`
    summed over the tokens (``reduction="sum"``) or averaged over those that
    count (``"mean"``; 0 when none does), a 0-dimensional float32 tensor, and
    the gradients of ``grad_scale`` times it, of x's type.

    Between the products, exponentials are held as float16 (within 2^-11 of the
    value, or 2^-40 of the largest among some neighbouring words) and
    probabilities minus the one-hot in the operands' type, each before the
    gradients' own rounding.  They take up to 1 GiB (and the rows' padding; more
    where 256 tokens do), and more tokens run in pieces.  float16 gradients of a
    mean over many tokens reach the type's subnormals: scale them
    (``grad_scale``) as loss scaling does."""
    if reduction in ("mean", "sum"):
        r = _fast("linear_cross_entropy_grad", x, weight, targets, ignore_index, reduction == "mean",
                  grad_scale)
        if r is not None:
            return r
    torch = _torch()
    if reduction not in ("mean", "sum"):
        raise LaunchError(f"unknown reduction {reduction!r}; expected 'mean' or 'sum'")
    index, code, rows, w, ids, size, ignore = _head_args(torch, x, weight, targets, ignore_index)
    n, width = rows.shape
    vocab = w.shape[0]
    device = x.device
    loss = torch.empty((), dtype=torch.float32, device=device)
    dx = torch.empty(x.shape, dtype=x.dtype, device=device)
    dweight = torch.empty((vocab, width), dtype=x.dtype, device=device)
    lib = _native.lib()
    need = lib.hcg_linear_cross_entropy_workspace(n, vocab, width, _ptr(w), _ld(w), 1)
    ws = _workspace(torch, need, device)
    _call(torch, index, lib.hcg_linear_cross_entropy_grad, "hcg_linear_cross_entropy_grad", code, _ptr(rows),
          _ld(rows), n, _ptr(w), _ld(w), vocab, width, size, _ptr(ids), ignore, reduction == "mean", grad_scale,
          _ptr(loss), _ptr(dx), width, _ptr(dweight), width, _ptr(ws), need)
    return loss, dx, dweight
