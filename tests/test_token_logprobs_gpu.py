"""`glue.token_logprobs` against log-softmax in 64 bits; tokens have to be equal.

What may differ, relative to l = sum e^(x - m): 2^-22 for the exponential, 2^-23 a unit of |x - m|
for its argument (17 units at most on the average over a vocabulary of 2^17), 2^-24 an addition
(a thread's own, one in 512 of the row's at most, and some 64 joining threads and blocks); and the
rounding of the result.  The entropy's second term is such a sum too, up to ln(vocab) times l."""

from __future__ import annotations

import math

import pytest
import torch

from linnet_b200 import glue

pytestmark = pytest.mark.gpu


def _want(logits, tokens, top):
    x = logits.double()
    below = x - x.amax(dim=-1, keepdim=True)  # first: at 10^38 even 64 bits hold no ln l beside the logits
    logprob = below - below.exp().sum(dim=-1, keepdim=True).log()
    p = logprob.exp()
    entropy = -torch.where(p > 0, p * logprob, torch.zeros_like(p)).sum(dim=-1)
    given = logprob.gather(1, tokens.clamp_min(0)[:, None])[:, 0]
    given = torch.where(tokens < 0, torch.zeros_like(given), given)
    index = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return given, entropy, logprob.gather(1, index), index


def _check(logits, tokens, top):
    got = glue.token_logprobs(logits, tokens, top)
    given, entropy, best, index = _want(logits, tokens, top)
    vocab = logits.shape[1]
    sums = 2.0 ** -22 + 17 * 2.0 ** -23 + (vocab / 512 + 64) * 2.0 ** -24
    for mine, exact, scale in ((got.logprob, given, 1.0), (got.entropy, entropy, 1.0 + 2 * math.log(vocab + 1)), (got.top_logprobs, best, 1.0)):
        assert mine.dtype == torch.float32 and mine.shape == exact.shape
        finite = torch.isfinite(exact)
        assert torch.equal(mine[~finite].double().nan_to_num(nan=5e30), exact[~finite].nan_to_num(nan=5e30))
        off = (mine.double() - exact)[finite].abs()
        assert bool((off <= scale * sums + exact[finite].abs() * 2.0 ** -23).all()), float(off.max())
    assert got.top_tokens.dtype == torch.int64 and torch.equal(got.top_tokens, index)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 128256, 20), (1, 1, 1), (1, 1, 0), (2, 7, 7), (5, 33, 32), (3, 255, 5), (3, 257, 20), (64, 32000, 20), (700, 4099, 1),
    (17, 128257, 0), (600, 1000, 32), (9, 50001, 32), (149, 16384, 6)])
def test_token_logprobs(dtype, rows, vocab, top):
    gen = torch.Generator(device="cuda").manual_seed(vocab + top)
    logits = (torch.randn(rows, vocab, device="cuda", generator=gen) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    tokens[rows // 2] = vocab - 1
    _check(logits, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["equal", "levels", "steps", "one above", "rising", "falling", "zeros of both signs", "crowded"])
def test_ties_go_to_the_lowest_index(dtype, kind):
    vocab = 40000
    i = torch.arange(vocab, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows = {
        "equal": torch.zeros(vocab, device="cuda"),
        "levels": torch.randint(0, 4, (vocab,), device="cuda", generator=gen).float(),
        "steps": (i // 300).float() / 8,
        "one above": torch.where(i == 31234, 1.0, 0.0),
        "rising": i.float() / vocab,
        "falling": -i.float() / vocab,
        "zeros of both signs": torch.where(i % 3 == 0, 0.0, -0.0),
        "crowded": torch.where(i // 256 == 77, 9.0 + (i % 256).float() / 32, torch.rand(vocab, device="cuda", generator=gen)),
    }[kind]
    logits = torch.stack([rows, rows.flip(0), rows * 0.5]).to(dtype)
    for top in (1, 20, 32):
        _check(logits, torch.tensor([0, 39999, 17], device="cuda"), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_logits(dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    vocab, lowest = 33333, torch.finfo(dtype).min
    logits = torch.randn(8, vocab, device="cuda", generator=gen).to(dtype)
    logits[0, 3:] = -math.inf                       # three tokens allowed: alternatives run into the forbidden ones
    logits[1, :] = -math.inf
    logits[1, 20000] = 1.0                          # one
    logits[2, :] = lowest                           # the type's lowest value everywhere: even odds
    logits[3, 5:] = lowest                          # ... behind a few real ones
    logits[4, :] = -math.inf                        # nothing allowed: no distribution, NaN
    logits[5, 1::2] = -math.inf
    logits[6, :] = torch.finfo(dtype).max           # the largest values
    logits[7, 100] = 60.0 if dtype != torch.float32 else 1e30  # far above the others
    tokens = torch.tensor([1, 20000, 7, 6, 0, 1, 5, 100], device="cuda")
    got = _check(logits[[0, 1, 2, 3, 5, 6, 7]], tokens[[0, 1, 2, 3, 5, 6, 7]], 20)
    assert float(got.logprob[1]) == 0.0 and float(got.entropy[1]) == 0.0
    nothing = glue.token_logprobs(logits[4:5], tokens[4:5], 20)
    assert bool(nothing.logprob.isnan().all()) and bool(nothing.entropy.isnan().all())
    assert torch.equal(nothing.top_tokens, torch.arange(20, device="cuda")[None])


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_nan_and_infinity_show(value):
    logits = torch.randn(3, 5000, device="cuda")
    logits[1, 4321] = value
    got = glue.token_logprobs(logits, torch.tensor([1, 2, 3], device="cuda"), 20)
    assert bool(got.logprob[1].isnan()) and bool(got.entropy[1].isnan()) and bool(got.top_logprobs[1].isnan().all())
    assert bool(torch.isfinite(got.logprob[[0, 2]]).all()) and bool(torch.isfinite(got.entropy[[0, 2]]).all())
    assert bool(((got.top_tokens >= 0) & (got.top_tokens < 5000)).all())
    logits[1, :] = value
    got = glue.token_logprobs(logits, torch.tensor([1, 2, 3], device="cuda"), 20)
    assert bool(got.logprob[1].isnan()) and bool(((got.top_tokens >= 0) & (got.top_tokens < 5000)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("begin,vocab,stride", [(0, 1001, 1003), (1, 1001, 1001), (3, 257, 264), (7, 4096, 5000), (5, 9, 16)])
def test_rows_at_any_address(dtype, begin, vocab, stride):
    """A part of a wider row (a vocabulary padded or split over ranks); NaN around it is never read into it."""
    gen = torch.Generator(device="cuda").manual_seed(begin)
    base = torch.full((6 * stride + begin,), math.nan, device="cuda", dtype=dtype)
    view = torch.as_strided(base, (5, vocab), (stride, 1), begin)
    view.copy_(torch.randn(5, vocab, device="cuda", generator=gen))
    _check(view, torch.randint(0, vocab, (5,), device="cuda", generator=gen), min(20, vocab))


def test_tokens_that_were_not_given_or_do_not_exist():
    logits = torch.randn(4, 1000, device="cuda")
    glue.decoder_status()
    got = glue.token_logprobs(logits, torch.tensor([3, -1, -100, 999], device="cuda"))
    assert float(got.logprob[1]) == 0.0 and float(got.logprob[2]) == 0.0 and float(got.logprob[0]) < 0.0
    assert got.top_tokens.shape == (4, 0) and got.top_logprobs.shape == (4, 0)
    glue.decoder_status()
    got = glue.token_logprobs(logits, torch.tensor([3, 1 << 40, 5, 1000], device="cuda"))
    assert bool(got.logprob[1].isnan()) and bool(got.logprob[3].isnan()) and bool(torch.isfinite(got.entropy).all())
    with pytest.raises(ValueError, match="row"):
        glue.decoder_status()
    glue.decoder_status()


def test_no_rows_one_row_many_times_and_refusals():
    empty = glue.token_logprobs(torch.empty(0, 10, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert empty.logprob.shape == (0,) and empty.top_tokens.shape == (0, 3)
    row = torch.randn(1, 3000, device="cuda").to(torch.bfloat16)
    _check(row.expand(70, -1), torch.arange(70, device="cuda"), 4)
    logits, tokens = torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="0 to 8"):
        glue.token_logprobs(logits, tokens, 9)
    with pytest.raises(ValueError, match="0 to 8"):
        glue.token_logprobs(logits, tokens, -1)
    with pytest.raises(ValueError, match="int64"):
        glue.token_logprobs(logits, tokens.int())
    with pytest.raises(ValueError, match="int64"):
        glue.token_logprobs(logits, tokens[:1])
    with pytest.raises(ValueError, match="rows, vocab"):
        glue.token_logprobs(logits[0], tokens)
    with pytest.raises(RuntimeError, match="types"):
        glue.token_logprobs(logits.double(), tokens)
    with pytest.raises(RuntimeError, match="last dimension"):
        glue.token_logprobs(logits.T, torch.zeros(8, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="no derivative"):
        glue.token_logprobs(logits.requires_grad_(), tokens)


def test_the_same_bits_every_time_and_in_a_graph():
    gen = torch.Generator(device="cuda").manual_seed(8)
    logits = torch.randint(0, 60, (40, 60000), device="cuda", generator=gen).to(torch.bfloat16)  # many ties
    tokens = torch.randint(0, 60000, (40,), device="cuda", generator=gen)
    first = glue.token_logprobs(logits, tokens, 20)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, glue.token_logprobs(logits, tokens, 20)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = glue.token_logprobs(logits, tokens, 20)
    logits.copy_(logits.flip(0))
    want = glue.token_logprobs(logits, tokens, 20)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
