"""hc.gfx950.embedding and its gradient: strided tables, and more tokens than
one launch takes with every type of id, a padding row and unknown tokens."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import hc.gfx950 as g  # noqa: E402
from hc._errors import LaunchError  # noqa: E402

from .test_lm_gpu import (BF16, DEV, E32, F16, F32, TINY, U, _close, _embedding_grad_want, _gen, _randn,  # noqa: E402
                          _twice)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_lookup_in_a_table_of_strided_columns(dtype):
    table = _randn(_gen(1), (40, 90), dtype)[::2, ::3]
    tokens = torch.tensor([3, 19, 20, 0, -1, 3], device=DEV)
    out = g.embedding(tokens, table, scale=0.75)
    known = torch.tensor([True, True, False, True, False, True], device=DEV)
    assert torch.equal(out[known], (table[tokens[known]].float() * 0.75).to(dtype))
    assert out[~known].isnan().all()


def _tokens(gen, n, vocab, spread):
    u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
    if spread == "even":
        return (u * vocab).long().clamp_(max=vocab - 1)
    if spread == "one":  # nearly all the same row
        return torch.where(u < 0.97, vocab // 2, (u * 31337).long() % vocab)
    return ((torch.exp(u * math.log(vocab + 1.0)) - 1).long() * 7919 % vocab).clamp_(0, vocab - 1)


# Three launches (rows of more than 256 items, or more than 4096 tokens), and
# four past 8192 tokens; vocabularies below 64, that 64 ranges do not divide,
# and whose last range is nearly empty.
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,vocab,width,spread", [
    (100, 30, 2060, "one"), (5000, 1000, 40, "zipf"), (8192, 4097, 33, "zipf"), (8193, 5, 24, "even"),
    (8193, 4097, 130, "zipf"), (9000, 1, 9, "even"), (12000, 37, 515, "one"), (40000, 70001, 24, "zipf"),
    (40001, 4161, 64, "one"), (33000, 100, 16, "even"), (20000, 262147, 8, "even")])
@pytest.mark.parametrize("padding", [False, True])
def test_gradient_of_many_tokens(n, vocab, width, spread, ids, padding):
    gen = _gen(n + vocab)
    tokens = _tokens(gen, n, vocab, spread)
    # unknown tokens on both sides, at the batch's ends and inside it
    odd = torch.rand((n,), generator=gen, device=DEV)
    tokens = torch.where(odd < 0.05, -1 - tokens % 7, torch.where(odd > 0.95, vocab + tokens % 11, tokens))
    tokens[0], tokens[-1] = -(2**31), 2**31 - 1
    pad = None
    dy = _randn(gen, (n, width), BF16)
    dy[(tokens < 0) | (tokens >= vocab)] = float("nan")  # (they reach no row)
    if padding:
        pad = int(tokens[(tokens >= 0) & (tokens < vocab)].mode().values)
        dy[tokens == pad] = float("inf")
    tokens = tokens.to(ids)
    for out_dtype in (BF16, F32):
        got = _twice(lambda: g.embedding_grad(dy, tokens, vocab, scale=0.5, padding_idx=pad, dtype=out_dtype))
        want, mag, count = _embedding_grad_want(dy, tokens, vocab, 0.5, pad)
        _close(got, want, (count + 2) * E32 * mag + U[out_dtype] * want.abs() + TINY[out_dtype])
        assert (got[count[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("n,vocab", [(300, 64), (5000, 900), (9000, 900)])
def test_gradient_of_unknown_tokens_only(n, vocab):
    dy = torch.full((n, 48), float("nan"), device=DEV)
    tokens = torch.full((n,), -1, dtype=torch.int64, device=DEV)
    tokens[::2] = vocab
    assert (g.embedding_grad(dy, tokens, vocab) == 0).all()
    tokens[:] = 5
    assert (g.embedding_grad(dy, tokens, vocab, padding_idx=5) == 0).all()


def test_gradient_refuses_counts_that_are_no_whole_numbers():
    dy, tokens = torch.ones((3, 8), device=DEV), torch.tensor([0, 1, 4], device=DEV)
    for bad in (4.5, "5", None, float("inf"), float("nan")):
        with pytest.raises(LaunchError, match="vocab must be a whole number"):
            g.embedding_grad(dy, tokens, bad)
        if bad is not None:
            with pytest.raises(LaunchError, match="padding_idx must be a whole number"):
                g.embedding_grad(dy, tokens, 5, padding_idx=bad)
    want = g.embedding_grad(dy, tokens, 5)
    assert torch.equal(g.embedding_grad(dy, tokens, 5.0), want)
    assert torch.equal(g.embedding_grad(dy, tokens, torch.tensor(5), padding_idx=torch.tensor(2)), want)
