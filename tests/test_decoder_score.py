"""`Int4Decoder.score` at its edges, on the plain route and on the fused one: tokens past the vocabulary,
none given, equal logits, forbidden tokens, and what is refused.  `step` is replaced by one that
returns given logits, so that both routes have the same."""

from __future__ import annotations

import math

import pytest
import torch

from linnet_b200 import decoder as dec
from linnet_b200 import glue
from tests import decoder_util as du

VOCAB = dec.DecoderConfig.tiny().vocab


def scorer(logits: torch.Tensor, fused: bool) -> dec.Int4Decoder:
    cfg = dec.DecoderConfig.tiny()
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear)
    model.fused = fused
    model.step = lambda tokens, positions: logits
    return model


def rows() -> torch.Tensor:
    """Logits of few different values (so that most have equals), one row of one value, one row with
    most tokens forbidden, one with all of them, one that holds NaN."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randint(-4, 5, (7, VOCAB), generator=gen).to(torch.bfloat16)
    logits[1] = 0.5
    logits[2, torch.rand(VOCAB, generator=gen) < 0.97] = -math.inf
    logits[3] = -math.inf
    logits[4, 100] = math.nan
    logits[5, ::2] = -0.0
    logits[5, 1::2] = 0.0
    return logits


GIVEN = [3, VOCAB, 7, 1, -1, VOCAB - 1, 1 << 40]


def check(got: glue.TokenLogprobs, logits: torch.Tensor, top: int) -> None:
    """f32 sums of VOCAB terms: VOCAB * 2^-24 relative at the worst, and as much of numbers below 16."""
    logits = logits.double().cpu()
    want = logits - torch.logsumexp(logits, dim=-1, keepdim=True)
    given = torch.tensor(GIVEN)
    logprob = want.gather(1, given.clamp(0, VOCAB - 1)[:, None])[:, 0]
    logprob[given >= VOCAB], logprob[given < 0] = math.nan, 0.0
    near = dict(rtol=VOCAB * 2.0 ** -24, atol=16 * VOCAB * 2.0 ** -24, equal_nan=True)
    torch.testing.assert_close(got.logprob.double().cpu(), logprob, **near)
    entropy = -torch.special.xlogy(want.exp(), want.exp()).sum(dim=-1)
    torch.testing.assert_close(got.entropy.double().cpu(), entropy, **near)
    order = torch.tensor([sorted(range(VOCAB), key=lambda i: (-row[i], i))[:top] for row in logits.nan_to_num(nan=-math.inf).tolist()]).long()
    plain = [r for r in range(len(GIVEN)) if r != 4]  # where NaN stands in the order is not said
    assert torch.equal(got.top_tokens.cpu()[plain], order[plain])
    torch.testing.assert_close(got.top_logprobs.double().cpu()[plain], want.gather(1, order)[plain], **near)
    assert bool(got.top_logprobs[4].isnan().all())


def run(fused: bool, device: str, top: int) -> None:
    logits = rows().to(device)
    at = torch.zeros(len(GIVEN), dtype=torch.long, device=device)
    check(scorer(logits, fused).score(at, at, torch.tensor(GIVEN, device=device), top=top), logits, top)


@pytest.mark.parametrize("top", [0, 1, 5, 32, VOCAB])
def test_edges_of_the_plain_route(top):
    run(False, "cpu", top)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_edges_on_a_gpu(fused):
    for top in (0, 1, 5, 32):
        run(fused, "cuda", top)
    if fused:
        with pytest.raises(ValueError, match="batch row"):
            glue.decoder_status()
    glue.decoder_status()


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("given", [torch.tensor([1]), torch.tensor([[1, 2]]), torch.tensor([1, 2], dtype=torch.int32)])
def test_tokens_that_are_refused(given, fused):
    """Before the step: the caches are not written for a call that fails."""
    model = scorer(torch.zeros(2, VOCAB), fused)
    model.step = None
    with pytest.raises(ValueError, match="given"):
        model.score(torch.zeros(2, dtype=torch.long), torch.zeros(2, dtype=torch.long), given)


@pytest.mark.parametrize("top", [-1, VOCAB + 1])
def test_alternatives_that_are_refused(top):
    at = torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="alternatives"):
        scorer(torch.zeros(2, VOCAB), False).score(at, at, at, top=top)


# ---- every step of sampled answers, by itself ----------------------------------------------------

STEPS, BATCH = 6, 6


def _model(fused: bool) -> dec.Int4Decoder:
    device, linear = "cpu", du.oracle_linear
    if fused:
        from linnet_b200 import kernels

        device, linear = "cuda", kernels.int4_linear
    cfg = dec.DecoderConfig.tiny()
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, linear, device=device)
    model.fused = fused
    return model


def _furthest(model: dec.Int4Decoder, prompt: list[int], planted: int | None = None) -> list[float]:
    """How far each step's log probabilities of answers that share the prompt (of the token given and of
    eight alternatives, the worst of all rows) are from those of rows that step through prompt and answer
    by themselves on the plain route, as a share of what is allowed.  Two routes' logits differ by 3 % of
    the largest (`tests/test_decoder_shared.py`), a logit less the logarithm of a sum by twice that.
    `planted`: at this step the prompt is taken for one position shorter."""
    device = model.embed.device
    gen = torch.Generator().manual_seed(23)
    chosen = torch.randint(0, VOCAB, (STEPS + 1, BATCH), generator=gen)
    plain = _model(False)
    plain.allocate_cache(BATCH)
    sequence = [torch.full((BATCH,), token) for token in prompt] + list(chosen)
    want = []
    for at, token in enumerate(sequence[:-1]):
        logits = plain.step(token, torch.full((BATCH,), at)).double()
        if at >= len(prompt):
            want.append((torch.log_softmax(logits, dim=-1), 2 * 3e-2 * logits.abs().max().item()))
    model.allocate_cache(1)
    for at, token in enumerate(prompt):
        model.step(torch.tensor([token], device=device), torch.tensor([at], device=device))
    model.share_prefix(len(prompt), BATCH, STEPS)
    out = []
    for t, (exact, allowed) in enumerate(want):
        model.prefix_length.fill_(len(prompt) - (t == planted))
        got = model.score(chosen[t].to(device), torch.full((BATCH,), t, device=device), chosen[t + 1].to(device), top=8)
        tokens = torch.cat([chosen[t + 1][:, None], got.top_tokens.cpu()], dim=1)
        mine = torch.cat([got.logprob[:, None], got.top_logprobs], dim=1).double().cpu()
        out.append((mine - exact.gather(1, tokens)).abs().max().item() / allowed)
    return out


PROMPTS = [[7, 301, 12, 44, 44, 9, 250], [(i * 97) % VOCAB for i in range(25)]]


@pytest.mark.parametrize("prompt", PROMPTS, ids=["short", "longer"])
def test_every_step_of_the_plain_route(prompt):
    assert max(_furthest(_model(False), prompt)) <= 1.0


def test_a_step_at_the_wrong_position_shows():
    """A test of the tests around it."""
    share = _furthest(_model(False), PROMPTS[0], planted=3)
    assert max(share[:3]) <= 1.0 < share[3]


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", PROMPTS, ids=["short", "longer"])
def test_every_step_of_the_fused_route(prompt):
    assert max(_furthest(_model(True), prompt)) <= 1.0
    glue.decoder_status()
