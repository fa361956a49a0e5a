"""The two ends of a language model and the norm between them, as timed cases.

Three operators, each with its gradient: the embedding lookup with scaling,
layer norm, and the softmax cross entropy of a linear head over a vocabulary.
A case is one pass through one of them.  ``run`` computes it in plain torch
operations in 32 bits, or, with ``own`` set, by the framework's entry points
in ``hc.gfx950``; ``exact`` computes the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
IGNORE = -100
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
_MAX_LOSS = 8192 * 65536 * 4096  # tokens * vocabulary * width of the largest listed loss
_MAX_ELEMENTS = 1 << 27          # of the largest drawn activation or table


def _loss(name, path, tokens, vocab, width, dtype, ignored):
    return {"name": name, "path": path, "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype,
            "ignored": ignored}


def _norm(name, path, rows, width, dtype):
    return {"name": name, "path": path, "rows": rows, "width": width, "dtype": dtype}


def _embed(name, path, tokens, vocab, width, dtype):
    return {"name": name, "path": path, "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype}


def listed():
    return [
        # The head of a small model on a short batch: a character or byte-pair
        # vocabulary, where launches count.
        _loss("loss_grad_256x4096x512_f16", "loss_grad", 256, 4096, 512, "float16", 0.0),
        # An ordinary training step's head.
        _loss("loss_grad_8192x32768x2048_bf16", "loss_grad", 8192, 32768, 2048, "bfloat16", 0.0),
        # The largest: a wide model over a large vocabulary.
        _loss("loss_grad_8192x65536x4096_bf16", "loss_grad", 8192, 65536, 4096, "bfloat16", 0.0),
        # Fine-tuning on ragged batches: prompts and padding (a third of the
        # tokens) do not count, and no size is a multiple of anything.
        _loss("loss_grad_1999x50021x1027_f16", "loss_grad", 1999, 50021, 1027, "float16", 0.35),
        # Scoring a few candidate tokens while serving: bound by reading the
        # head's weights.
        _loss("loss_16x65536x4096_bf16", "loss", 16, 65536, 4096, "bfloat16", 0.0),
        # One token's norm while decoding: the smallest call.
        _norm("norm_1x4096_bf16", "norm", 1, 4096, "bfloat16"),
        # A training batch's norm, and its backward pass.
        _norm("norm_8192x4096_bf16", "norm", 8192, 4096, "bfloat16"),
        _norm("norm_grad_8192x4096_bf16", "norm_grad", 8192, 4096, "bfloat16"),
        # The same in 32 bits on odd sizes.
        _norm("norm_grad_3001x1027_f32", "norm_grad", 3001, 1027, "float32"),
        # A training batch's rows from a large table, and the table's gradient
        # (natural text: a few tokens fill much of the batch, most of the
        # table gets nothing).
        _embed("embed_8192x4096_of_65536_bf16", "embed", 8192, 65536, 4096, "bfloat16"),
        _embed("embed_grad_8192x4096_of_65536_bf16", "embed_grad", 8192, 65536, 4096, "bfloat16"),
        # A small model's table in 32 bits, odd sizes.
        _embed("embed_grad_999x515_of_5003_f32", "embed_grad", 999, 5003, 515, "float32"),
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
    path = rng.choice(["loss_grad", "loss_grad", "loss_grad", "loss", "norm", "norm_grad", "embed", "embed_grad"])
    if path in ("loss", "loss_grad"):
        tokens, vocab, width = _size(rng, 1, 16384), _size(rng, 256, 131072), _size(rng, 64, 8192)
        while tokens * vocab * width > _MAX_LOSS or vocab * width > 1 << 29:
            tokens, vocab = tokens // 2 | 1, max(256, vocab // 2 | 1)
        return {"path": path, "tokens": tokens, "vocab": vocab, "width": width,
                "dtype": rng.choice(["float16", "bfloat16"]), "ignored": rng.choice([0.0, 0.0, 0.1, 0.5, 0.9])}
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    if path in ("norm", "norm_grad"):
        rows, width = _size(rng, 1, 65536), _size(rng, 64, 16384)
        while rows * width > _MAX_ELEMENTS:
            rows = rows // 2 | 1
        return {"path": path, "rows": rows, "width": width, "dtype": dtype}
    tokens, vocab, width = _size(rng, 1, 65536), _size(rng, 128, 131072), _size(rng, 64, 8192)
    while max(tokens, vocab) * width > _MAX_ELEMENTS:
        tokens, vocab = tokens // 2 | 1, max(128, vocab // 2 | 1)
    return {"path": path, "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype}


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std + mean).to(dtype)


def _text(gen, tokens, vocab):
    """Token ids as text has them: the r-th most frequent about 1/r as often
    as the first, in an order of ids that has nothing to do with frequency."""
    u = torch.rand((tokens,), generator=gen, device=DEV, dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device=DEV)[rank]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = _generator(seed)
    dt, width = _DTYPES[case["dtype"]], case["width"]
    path = case["path"]
    if path in ("loss", "loss_grad"):
        tokens, vocab = case["tokens"], case["vocab"]
        weight = _normal(gen, (vocab, width), dt, 0.02)
        targets = _text(gen, tokens, vocab)
        # Hidden states after a norm; a trained head gives the target up to 12
        # more than a random word.
        lift = torch.rand((tokens, 1), generator=gen, device=DEV) * (12.0 / (0.02 * 0.02 * width))
        x = (torch.randn((tokens, width), generator=gen, device=DEV) + lift * weight[targets].float()).to(dt)
        drop = torch.rand((tokens,), generator=gen, device=DEV) < case["ignored"]
        return {"x": x, "weight": weight, "targets": torch.where(drop, IGNORE, targets)}
    if path in ("norm", "norm_grad"):
        rows = case["rows"]
        x = _normal(gen, (rows, width), dt, 1.5, 0.25)
        weight = _normal(gen, (width,), dt, 0.1, 1.0)
        bias = _normal(gen, (width,), dt, 0.1)
        if path == "norm":
            return {"x": x, "weight": weight, "bias": bias}
        # What the forward pass left behind.
        xf = x.double()
        mean = xf.mean(1)
        rstd = 1.0 / torch.sqrt((xf - mean[:, None]).square().mean(1) + 1e-5)
        return {"x": x, "weight": weight, "mean": mean.float(), "rstd": rstd.float(),
                "dy": _normal(gen, (rows, width), dt)}
    tokens, vocab = case["tokens"], case["vocab"]
    ids = _text(gen, tokens, vocab)
    if path == "embed":
        return {"tokens": ids, "table": _normal(gen, (vocab, width), dt, 0.02), "scale": math.sqrt(width)}
    return {"tokens": ids, "dy": _normal(gen, (tokens, width), dt), "vocab": vocab, "scale": math.sqrt(width)}


def prepare(case, seed):
    return {"path": case["path"], "dtype": _DTYPES[case["dtype"]], **_inputs(case, seed)}


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
    path = s["path"]
    if path == "loss_grad":
        return g.linear_cross_entropy_grad(s["x"], s["weight"], s["targets"])
    if path == "loss":
        return g.linear_cross_entropy(s["x"], s["weight"], s["targets"])
    if path == "norm":
        return g.layer_norm(s["x"], s["weight"], s["bias"])
    if path == "norm_grad":
        return g.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if path == "embed":
        return g.embedding(s["tokens"], s["table"], scale=s["scale"])
    return g.embedding_grad(s["dy"], s["tokens"], s["vocab"], scale=s["scale"])


def _run_plain(s):
    path, dt = s["path"], s["dtype"]
    if path in ("loss", "loss_grad"):
        x, weight, targets = s["x"].float(), s["weight"].float(), s["targets"]
        live = targets != IGNORE
        at = torch.where(live, targets, 0)[:, None]
        logits = x @ weight.t()
        top = logits.amax(1, keepdim=True)
        e = torch.exp(logits - top)
        total = e.sum(1, keepdim=True)
        lse = (top + torch.log(total))[:, 0]
        loss = torch.where(live, lse - logits.gather(1, at)[:, 0], 0.0)
        if path == "loss":
            return loss, torch.where(live, lse, 0.0)
        count = live.sum().clamp(min=1)
        share = live[:, None] / count
        g = e * (share / total)
        g.scatter_add_(1, at, -share)
        return loss.sum() / count, (g @ weight).to(dt), (g.t() @ x).to(dt)
    if path == "norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        centred = x - mean
        rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + 1e-5)
        y = centred * rstd * s["weight"].float() + s["bias"].float()
        return y.to(dt), mean[:, 0], rstd[:, 0]
    if path == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        gw = dy * s["weight"].float()
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
        return dx.to(dt), (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)
    if path == "embed":
        return (s["table"][s["tokens"]].float() * s["scale"]).to(dt)
    dy = s["dy"].float() * s["scale"]
    grad = torch.zeros((s["vocab"], dy.shape[1]), dtype=torch.float32, device=dy.device)
    return grad.index_add_(0, s["tokens"], dy).to(dt)


def work(case):
    size, width = _BYTES[case["dtype"]], case["width"]
    path = case["path"]
    if path in ("loss", "loss_grad"):
        tokens, vocab = case["tokens"], case["vocab"]
        # Hidden states, weights and targets in (ids are 64-bit); losses, or
        # the loss and both gradients, out.  Tokens that do not count need no
        # product.
        live = max(1.0, tokens * (1.0 - case["ignored"]))
        read = size * (tokens + vocab) * width + 8 * tokens
        if path == "loss":
            return {"bytes": read + 8 * tokens, "flops": 2 * live * vocab * width}
        return {"bytes": read + size * (tokens + vocab) * width, "flops": 6 * live * vocab * width}
    if path in ("norm", "norm_grad"):
        rows = case["rows"]
        if path == "norm":
            return {"bytes": 2 * size * rows * width + 2 * size * width + 8 * rows, "flops": 8 * rows * width}
        return {"bytes": 3 * size * rows * width + 3 * size * width + 8 * rows, "flops": 14 * rows * width}
    tokens, vocab = case["tokens"], case["vocab"]
    if path == "embed":
        # (Rows that several tokens name are counted once at most per token.)
        return {"bytes": 8 * tokens + size * width * (min(tokens, vocab) + tokens), "flops": tokens * width}
    return {"bytes": 8 * tokens + size * width * (tokens + vocab), "flops": 2 * tokens * width}


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits."""
    t = _inputs(case, seed)
    path = case["path"]
    if path in ("loss", "loss_grad"):
        if case["tokens"] * case["vocab"] > 1 << 30:
            return None  # (the probabilities alone would take over 8 GiB several times)
        x, w, y = t["x"].double(), t["weight"].double(), t["targets"]
        keep = torch.nonzero(y != IGNORE)[:, 0]
        xk, yk = x[keep], y[keep]
        z = torch.mm(xk, w.t().contiguous())
        lse_k = torch.logsumexp(z, 1)
        loss_k = lse_k - z[torch.arange(len(keep), device=DEV), yk]
        n = case["tokens"]
        if path == "loss":
            return (torch.zeros(n, dtype=torch.float64, device=DEV).index_copy_(0, keep, loss_k),
                    torch.zeros(n, dtype=torch.float64, device=DEV).index_copy_(0, keep, lse_k))
        count = max(1, len(keep))
        z -= lse_k[:, None]
        p = z.exp_()
        p[torch.arange(len(keep), device=DEV), yk] -= 1.0
        p /= count
        dx = torch.zeros((n, case["width"]), dtype=torch.float64, device=DEV)
        dx[keep] = torch.mm(p, w)
        return loss_k.sum() / count, dx, torch.mm(p.t().contiguous(), xk)
    if path == "norm":
        x = t["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + 1e-5).pow(-0.5)
        return (x - mean[:, None]) * rstd[:, None] * t["weight"].double() + t["bias"].double(), mean, rstd
    if path == "norm_grad":
        x, dy, w = t["x"].double(), t["dy"].double(), t["weight"].double()
        mean, rstd = t["mean"].double()[:, None], t["rstd"].double()[:, None]
        d = case["width"]
        xhat = (x - mean) * rstd
        c1 = (dy * w).sum(1, keepdim=True)
        c2 = (dy * w * xhat).sum(1, keepdim=True)
        return (rstd / d) * (d * dy * w - c1 - xhat * c2), (dy * xhat).sum(0), dy.sum(0)
    if path == "embed":
        return t["table"].double()[t["tokens"]] * t["scale"]
    order = torch.argsort(t["tokens"], stable=True)
    out = torch.zeros((case["vocab"], case["width"]), dtype=torch.float64, device=DEV)
    return out.index_put_((t["tokens"][order],), t["dy"].double()[order] * t["scale"], accumulate=True)
