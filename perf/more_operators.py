"""Linear layers in 8-bit floating point, and the norm that feeds them, as timed cases.

Four operators: the root-mean-square norm with the residual's addition, in
16 or 32 bits or in 8 bits with a scale for each 128 columns; its gradient; the
quantiser of matrices, by rows of 128 or tiles of 128 x 128, also transposed;
and the product of two quantised matrices.  A case is one pass through one of
them.  ``run`` computes it in plain torch operations in 32 bits, or, with
``own`` set, by the framework's entry points in ``hc.gfx950``; ``exact``
computes the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128   # elements that share a scale
EPS = 1e-6
SMALL = 2.0**-100  # the least maximum that a block is scaled by
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32,
           "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2, "e8m0": torch.float8_e8m0fnu}
_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4, "e8m0": 1}
_LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
_MAX_PRODUCT = 8192**3           # tokens * outputs * inputs of the largest listed product
_MAX_ELEMENTS = 1 << 26          # of the largest drawn activation or weight


def _norm(name, path, rows, width, dtype, residual, to="e4m3", scale="float32"):
    case = {"name": name, "path": path, "rows": rows, "width": width, "dtype": dtype, "residual": residual}
    return {**case, "to": to, "scale": scale} if path == "norm_fp8" else case


def _quantize(name, rows, cols, dtype, block, transpose, to, scale):
    return {"name": name, "path": "quantize", "rows": rows, "cols": cols, "dtype": dtype, "block": block,
            "transpose": transpose, "to": to, "scale": scale}


def _linear(name, tokens, outputs, inputs, x="e4m3", block="tile", scale="float32", out="bfloat16"):
    return {"name": name, "path": "linear", "tokens": tokens, "outputs": outputs, "inputs": inputs, "x": x,
            "block": block, "scale": scale, "out": out}


def listed():
    return [
        # One token's norm before an 8-bit layer while decoding: the smallest
        # call, all latency.
        _norm("norm_fp8_1x4096_bf16", "norm_fp8", 1, 4096, "bfloat16", "bfloat16"),
        # A training batch's, or a long prompt's.
        _norm("norm_fp8_8192x4096_bf16", "norm_fp8", 8192, 4096, "bfloat16", "bfloat16"),
        # The same before a 16-bit layer, with the residual kept in 32 bits.
        _norm("norm_8192x4096_f16_f32", "norm", 8192, 4096, "float16", "float32"),
        # Its backward pass in training, with the residual path's gradient.
        _norm("norm_grad_8192x4096_bf16", "norm_grad", 8192, 4096, "bfloat16", "bfloat16"),
        # And in 32 bits on odd sizes.
        _norm("norm_grad_3001x1027_f32", "norm_grad", 3001, 1027, "float32", "float32"),
        # A batch's output gradient, quantised along the tokens for the weight's
        # gradient: read by rows, written transposed.
        _quantize("quantize_8192x4096_bf16_t_e5m2", 8192, 4096, "bfloat16", "row", True, "e5m2", "float32"),
        # A weight's 32-bit master copy into tiles, once per training step.
        _quantize("quantize_8192x8192_f32_tile", 8192, 8192, "float32", "tile", False, "e4m3", "float32"),
        # One token through a layer: bound by reading the weight.
        _linear("linear_1x8192x8192", 1, 8192, 8192),
        # An ordinary layer of a training step or a prompt.
        _linear("linear_4096x4096x4096", 4096, 4096, 4096),
        # The largest, with scales that are powers of two.
        _linear("linear_8192x8192x8192_e8m0", 8192, 8192, 8192, scale="e8m0"),
        # No size a multiple of anything.
        _linear("linear_4095x3001x1027_f16", 4095, 3001, 1027, out="float16"),
        # A weight's gradient over a batch of 8192 tokens: both operands scaled
        # by rows, output gradients in e5m2, 32 bits out.
        _linear("linear_dw_4096x4096x8192_f32", 4096, 4096, 8192, x="e5m2", block="row", out="float32"),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]: a third of them odd, a third odd multiples of
    8, a third powers of two."""
    v = lo * (hi / lo) ** rng.random()
    kind = rng.randrange(3)
    if kind == 0:
        v = int(v) | 1
    elif kind == 1:
        v = (int(v / 8) | 1) * 8
    else:
        v = 2 ** round(math.log2(v))
    return min(hi, max(lo, v))


def draw(rng):
    path = rng.choice(["linear", "linear", "linear", "linear", "norm", "norm_fp8", "norm_grad", "quantize"])
    scale, to = rng.choice(["float32", "float32", "e8m0"]), rng.choice(["e4m3", "e4m3", "e5m2"])
    if path == "linear":
        tokens, outputs, inputs = _size(rng, 1, 16384), _size(rng, 64, 16384), _size(rng, 64, 16384)
        while tokens * outputs * inputs > _MAX_PRODUCT or outputs * inputs > _MAX_ELEMENTS:
            tokens, outputs = tokens // 2 | 1, max(64, outputs // 2 | 1)
        return {"path": path, "tokens": tokens, "outputs": outputs, "inputs": inputs, "x": to,
                "block": rng.choice(["tile", "tile", "row"]), "scale": scale,
                "out": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    rows, width = _size(rng, 1, 65536), _size(rng, 64, 16384)
    while rows * width > _MAX_ELEMENTS // 2:
        rows = rows // 2 | 1
    if path == "quantize":
        return {"path": path, "rows": rows, "cols": width, "dtype": dtype, "block": rng.choice(["row", "row", "tile"]),
                "transpose": rng.choice([False, True]), "to": to, "scale": scale}
    case = {"path": path, "rows": rows, "width": width, "dtype": dtype,
            "residual": rng.choice([dtype, dtype, "float32"] if path == "norm_grad" else ["none", dtype, "float32"])}
    return {**case, "to": to, "scale": scale} if path == "norm_fp8" else case


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std + mean).to(dtype)


def _activation(gen, rows, width, dtype, std=1.0):
    """Hidden states: a few columns are much larger than the others."""
    loud = 1.0 + 15.0 * (torch.rand((width,), generator=gen, device=DEV) < 0.01)
    return (torch.randn((rows, width), generator=gen, device=DEV) * (std * loud)).to(dtype)


def _padded(q):
    """The matrix in rows of whole 16 bytes, as the quantiser leaves them."""
    rows, cols = q.shape
    held = torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.uint8, device=DEV)
    held[:, :cols] = q.view(torch.uint8)
    return held.view(q.dtype)[:, :cols]


def _blocks(x, block):
    """x in blocks: (row blocks, rows of one, column blocks, BLOCK), zeros past the ends."""
    rows, cols = x.shape
    high = BLOCK if block == "tile" else 1
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % high))
    return x.view(x.shape[0] // high, high, x.shape[1] // BLOCK, BLOCK)


def _quantized(x, block, to, scale):
    """(q, scale) of a float32 matrix in plain operations."""
    rows, cols = x.shape
    parts = _blocks(x, block)
    top = parts.abs().amax((1, 3)).clamp_(min=SMALL)
    largest = _LARGEST[to]
    if scale == "e8m0":
        mantissa, exponent = torch.frexp(top)
        power = exponent + (mantissa > 0.875) - int(math.log2(largest / 1.75)) - 1
        scales = torch.ldexp(torch.ones_like(top), power)
        inverse = torch.ldexp(torch.ones_like(top), -power)
    else:
        scales, inverse = top / largest, largest / top
    q = (parts * inverse[:, None, :, None]).flatten(2).flatten(0, 1)[:rows, :cols]
    return q.to(_DTYPES[to]), scales.to(_DTYPES[scale])


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    path = case["path"]
    if path == "linear":
        tokens, outputs, inputs = case["tokens"], case["outputs"], case["inputs"]
        if case["x"] == "e5m2":  # a gradient
            x = _activation(gen, tokens, inputs, torch.float32, 1e-3)
        else:
            x = _activation(gen, tokens, inputs, torch.float32)
        if case["block"] == "tile":
            weight = _normal(gen, (outputs, inputs), torch.float32, 0.02)
        else:
            weight = _activation(gen, outputs, inputs, torch.float32)
        qx, sx = _quantized(x, "row", case["x"], case["scale"])
        qw, sw = _quantized(weight, case["block"], "e4m3", case["scale"])
        # Scales lie block by block, as the quantiser leaves them.
        return {"x": _padded(qx), "sx": sx.t().contiguous().t(), "weight": _padded(qw), "sw": sw.t().contiguous().t()}
    dt = _DTYPES[case["dtype"]]
    if path == "quantize":
        if case["transpose"]:
            return {"x": _activation(gen, case["rows"], case["cols"], dt, 1e-3)}
        return {"x": _normal(gen, (case["rows"], case["cols"]), dt, 0.02)}
    rows, width = case["rows"], case["width"]
    weight = _normal(gen, (width,), dt, 0.1, 1.0)
    wide = None if case["residual"] == "none" else _DTYPES[case["residual"]]
    if path == "norm_grad":
        h = _activation(gen, rows, width, wide, 2.0)
        # What the forward pass left behind.
        rstd = (1.0 / torch.sqrt(h.double().square().mean(1) + EPS)).float()
        return {"dy": _normal(gen, (rows, width), dt), "h": h, "rstd": rstd, "weight": weight,
                "dresidual": _normal(gen, (rows, width), wide)}
    return {"x": _normal(gen, (rows, width), dt), "weight": weight,
            "residual": None if wide is None else _activation(gen, rows, width, wide, 2.0)}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


def _entry_points():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "5_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import hc.gfx950 as g

    return g


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    g = sys.modules.get("hc.gfx950") or _entry_points()
    c = s["case"]
    path = c["path"]
    if path == "linear":
        return g.linear_fp8(s["x"], s["sx"], s["weight"], s["sw"], out_dtype=_DTYPES[c["out"]])
    if path == "quantize":
        return g.quantize_fp8(s["x"], block=c["block"], transpose=c["transpose"], dtype=_DTYPES[c["to"]],
                              scale_dtype=_DTYPES[c["scale"]])
    if path == "norm_grad":
        return g.rms_norm_grad(s["dy"], s["h"], s["rstd"], s["weight"], dresidual=s["dresidual"])
    if path == "norm_fp8":
        return g.rms_norm_fp8(s["x"], s["weight"], s["residual"], eps=EPS, dtype=_DTYPES[c["to"]],
                              scale_dtype=_DTYPES[c["scale"]])
    return g.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)


def _plain_values(q, scale, block):
    """The float32 values that a quantised matrix stands for."""
    rows, cols = q.shape
    spread = _blocks(q.float(), block) * scale.float()[:, None, :, None]
    return spread.flatten(2).flatten(0, 1)[:rows, :cols]


def _run_plain(s):
    c = s["case"]
    path = c["path"]
    if path == "linear":
        x, w = _plain_values(s["x"], s["sx"], "row"), _plain_values(s["weight"], s["sw"], c["block"])
        return (x @ w.t()).to(_DTYPES[c["out"]])
    if path == "quantize":
        x = s["x"].float()
        return _quantized(x.t() if c["transpose"] else x, c["block"], c["to"], c["scale"])
    weight = s["weight"].float()
    if path == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = s["h"].float() * rstd
        gw = dy * weight
        dh = rstd * (gw - xhat * (gw * xhat).mean(1, keepdim=True)) + s["dresidual"].float()
        return dh.to(s["h"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype)
    x = s["x"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(s["residual"].dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(1) + EPS)
    y = hf * rstd[:, None] * weight
    if path == "norm":
        return y.to(x.dtype), h, rstd
    return (*_quantized(y, "row", c["to"], c["scale"]), h, rstd)


def work(case):
    path = case["path"]
    if path == "linear":
        t, v, k = case["tokens"], case["outputs"], case["inputs"]
        scales = -(-k // BLOCK) * (t + (-(-v // BLOCK) if case["block"] == "tile" else v))
        return {"bytes": (t + v) * k + scales * _BYTES[case["scale"]] + t * v * _BYTES[case["out"]],
                "flops": 2 * t * v * k}
    size = _BYTES[case["dtype"]]
    if path == "quantize":
        rows, cols = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        scales = -(-cols // BLOCK) * (-(-rows // BLOCK) if case["block"] == "tile" else rows)
        return {"bytes": rows * cols * (size + 1) + scales * _BYTES[case["scale"]], "flops": 3 * rows * cols}
    rows, width = case["rows"], case["width"]
    wide = _BYTES.get(case["residual"], 0)
    if path == "norm_grad":
        return {"bytes": rows * width * (size + 3 * wide) + 2 * size * width + 4 * rows, "flops": 9 * rows * width}
    result = {"bytes": rows * width * (size + 2 * wide) + size * width + 4 * rows, "flops": 5 * rows * width}
    if path == "norm":
        result["bytes"] += rows * width * size
    else:
        result["bytes"] += rows * (width + -(-width // BLOCK) * _BYTES[case["scale"]])
        result["flops"] += 3 * rows * width
    return result


def _exact_quantized(x, block, to, scale):
    """(q before its rounding, scale) in 64 bits; no q for e5m2, whose rounding
    alone is 5% of it."""
    rows, cols = x.shape
    up = -(-rows // BLOCK) if block == "tile" else rows
    across = -(-cols // BLOCK)
    top = torch.full((up, across), SMALL, dtype=torch.float64, device=DEV)
    for j in range(across):
        most = x[:, j * BLOCK:(j + 1) * BLOCK].abs().max(1).values
        if block == "tile":
            most = torch.stack([m.max() for m in most.split(BLOCK)])
        top[:, j] = torch.maximum(top[:, j], most)
    scales = top / _LARGEST[to]
    if scale == "e8m0":
        # the least power of two that is not below it
        power = torch.ceil(torch.log2(scales)) - 1.0
        power = torch.where(torch.exp2(power) < scales, power + 1.0, power)
        scales = torch.exp2(power)
    down = torch.arange(rows, device=DEV) // (BLOCK if block == "tile" else 1)
    if to == "e5m2":
        return None, scales
    return x / scales[down][:, torch.arange(cols, device=DEV) // BLOCK], scales


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits (8-bit values before
    their rounding)."""
    t = _inputs(case, seed)
    path = case["path"]
    if path == "linear":
        across = torch.arange(case["inputs"], device=DEV) // BLOCK
        down = torch.arange(case["outputs"], device=DEV) // (BLOCK if case["block"] == "tile" else 1)
        x = t["x"].double().mul_(t["sx"].double()[:, across])
        w = t["weight"].double().mul_(t["sw"].double()[down][:, across])
        return torch.mm(x, w.t().contiguous())
    if path == "quantize":
        x = t["x"].double()
        return _exact_quantized(x.t().contiguous() if case["transpose"] else x, case["block"], case["to"], case["scale"])
    w = t["weight"].double()
    if path == "norm_grad":
        dy, h, r = t["dy"].double(), t["h"].double(), t["rstd"].double()
        along = torch.einsum("ij,ij->i", dy * w, h) * r.pow(3) / case["width"]
        return t["dresidual"].double() + r[:, None] * dy * w - along[:, None] * h, torch.mv((dy * h).t().contiguous(), r)
    x = t["x"].double()
    h = x if t["residual"] is None else x + t["residual"].double()
    # (the norm is of the sum as it is held)
    held = h if t["residual"] is None else h.to(t["residual"].dtype).double()
    rstd = (torch.linalg.vector_norm(held, dim=1).square() / case["width"] + EPS).pow(-0.5)
    y = held * w * rstd[:, None]
    if path == "norm":
        return y, h, rstd
    return (*_exact_quantized(y, "row", case["to"], case["scale"]), h, rstd)
