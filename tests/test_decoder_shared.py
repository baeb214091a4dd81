"""Answers that share their prompt's cache (`Int4Decoder.share_prefix`) and the log probabilities of
their tokens (`Int4Decoder.score`): rotary positions, shared-prefix attention and token log
probabilities as one decode step uses them.  On the CPU the plain route with the oracle as the linear
operator; on a GPU the kernels against that route.

Tolerance of logits: a layer of these models rounds its activations to bf16 (by 2^-9 of the value at
most, half a step of 2^-8) about eight times on the way to the next, two layers and the head some 17
times, so that two routes whose sums differ in order come apart by 17 * 2 * 2^-9 = 6.6 % at the worst,
and by sqrt(34) * 2^-9 = 1.1 % where the roundings are independent: 3 % of the largest logit, as the
tests of the decoder's other routes have it."""

from __future__ import annotations

import dataclasses
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from linnet_b200 import decoder as dec
from linnet_b200.rope import RopeScaling
from tests import decoder_util as du
from tests.test_decoder import _free_port

LLAMA3 = RopeScaling("llama3", 4.0, original_positions=16)
YARN = RopeScaling("yarn", 8.0, original_positions=16)
PROMPT = [7, 301, 12, 44, 44, 9, 250]


def config(scaling=None) -> dec.DecoderConfig:
    return dataclasses.replace(dec.DecoderConfig.tiny(), rope_scaling=scaling)


def prefill(model, prompt, device="cpu") -> None:
    for at, token in enumerate(prompt):
        model.step(torch.tensor([token], device=device), torch.tensor([at], device=device))


def answers(cfg, batch: int, steps: int, device="cpu") -> torch.Tensor:
    gen = torch.Generator().manual_seed(11)
    return torch.randint(0, cfg.vocab, (steps, batch), generator=gen).to(device)


def shared_steps(model, cfg, prompt, tokens, device="cpu") -> torch.Tensor:
    """Logits [steps, batch, vocab] of rows that share the prompt's cache."""
    model.allocate_cache(1)
    prefill(model, prompt, device)
    steps, batch = tokens.shape
    model.share_prefix(len(prompt), batch, steps)
    return torch.stack([model.step(tokens[t], torch.full((batch,), t, device=device)) for t in range(steps)])


def copied_steps(model, cfg, prompt, tokens, device="cpu") -> torch.Tensor:
    """The same of rows that have each stepped through the prompt."""
    steps, batch = tokens.shape
    model.allocate_cache(batch)
    for at, token in enumerate(prompt):
        model.step(torch.full((batch,), token, device=device), torch.full((batch,), at, device=device))
    return torch.stack([model.step(tokens[t], torch.full((batch,), len(prompt) + t, device=device)) for t in range(steps)])


def close(got: torch.Tensor, want: torch.Tensor) -> None:
    got, want = got.float().cpu(), want.float().cpu()
    torch.testing.assert_close(got, want, rtol=3e-2, atol=3e-2 * want.abs().max().item())


@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN], ids=["plain", "llama3", "yarn"])
def test_rows_that_share_a_prompt_answer_as_rows_with_copies_of_it(scaling):
    cfg = config(scaling)
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear)
    tokens = answers(cfg, 3, 3)
    close(shared_steps(model, cfg, PROMPT, tokens), copied_steps(model, cfg, PROMPT, tokens))


def test_scaled_positions_change_the_answer():
    """A test of the test above: the scaling reaches the logits."""
    whole = du.whole_model(config())
    tokens = answers(config(), 2, 1)
    got = [shared_steps(du.rank_model(config(s), whole, 0, 1, du.oracle_linear), config(s), PROMPT, tokens).float()
           for s in (None, YARN)]
    assert (got[0] - got[1]).abs().max() > 0.1 * got[0].abs().max()


def test_the_caches_of_the_prompt_come_back():
    """After `end_prefix` the prompt's row is stepped on as if nothing had been shared; a prefix of no
    positions at all is one too; `allocate_cache` starts over."""
    cfg = config(LLAMA3)
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear)
    tokens = answers(cfg, 2, 2)
    before = shared_steps(model, cfg, PROMPT, tokens)
    kept = [c.clone() for c in model.prompt[0]]
    own = model.cache_k
    model.end_prefix()
    assert model.prefix is None and all(torch.equal(a, b) for a, b in zip(kept, model.cache_k))
    model.share_prefix(len(PROMPT), 2, 2)
    assert all(a is b for a, b in zip(own, model.cache_k))  # the same batch and room: the same caches
    again = torch.stack([model.step(tokens[t], torch.full((2,), t)) for t in range(2)])
    assert torch.equal(again, before)
    model.share_prefix(0, 2, 2)
    empty = model.step(tokens[0], torch.zeros(2, dtype=torch.long))
    model.allocate_cache(2)
    assert model.prefix is None and model.prompt is None
    close(empty, model.step(tokens[0], torch.zeros(2, dtype=torch.long)))


@pytest.mark.parametrize("arguments", [dict(length=33, batch=2, max_new=4), dict(length=-1, batch=2, max_new=4),
                                       dict(length=3, batch=0, max_new=4), dict(length=3, batch=2, max_new=0),
                                       dict(length=3, batch=2, max_new=4, row=1), dict(length=3, batch=2, max_new=4, row=-1)])
def test_a_prefix_that_is_not_there_is_refused(arguments):
    cfg = config()
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear)
    with pytest.raises(ValueError, match="share_prefix"):
        model.share_prefix(**arguments)  # no cache yet
    model.allocate_cache(1)
    with pytest.raises(ValueError, match="share_prefix"):
        model.share_prefix(**arguments)
    assert model.prefix is None and model.cache_k[0].shape[0] == 1


def test_scores_of_the_plain_route():
    cfg = config()
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear)
    tokens = answers(cfg, 3, 1)
    logits = copied_steps(model, cfg, PROMPT[:2], tokens)[0]
    given = torch.tensor([5, -1, 400])
    got = model.score(tokens[0], torch.full((3,), 2), given, top=4)  # the step again: it writes what is there
    want = torch.log_softmax(logits.double(), dim=-1)
    # f32 sums of 512 terms: 512 * 2^-24 relative at the worst
    torch.testing.assert_close(got.logprob.double(), torch.tensor([want[0, 5], 0.0, want[2, 400]]).double(), rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(got.entropy.double(), -(want.exp() * want).sum(-1), rtol=1e-4, atol=1e-4)
    best = want.topk(4, dim=-1)
    torch.testing.assert_close(got.top_logprobs.double(), best.values, rtol=1e-4, atol=1e-4)
    assert torch.equal(want.gather(1, got.top_tokens), best.values)


def _tp_worker(rank: int, world: int, port: int, out_dir: str) -> None:
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        cfg = config(LLAMA3)
        model = du.rank_model(cfg, du.whole_model(cfg), rank, world, du.oracle_linear)
        torch.save(shared_steps(model, cfg, PROMPT, answers(cfg, 2, 2)), os.path.join(out_dir, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_two_gloo_ranks_share_a_prompt(tmp_path):
    mp.spawn(_tp_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    cfg = config(LLAMA3)
    single = shared_steps(du.rank_model(cfg, du.whole_model(cfg), 0, 1, du.oracle_linear), cfg, PROMPT, answers(cfg, 2, 2))
    for rank in range(2):
        close(torch.load(tmp_path / f"rank{rank}.pt"), single)


# ---- on a GPU ---------------------------------------------------------------------------------


def gpu_model(cfg, whole=None, fused=True, fold=False):
    from linnet_b200 import kernels

    model = du.rank_model(cfg, whole or du.whole_model(cfg), 0, 1, kernels.int4_linear, device="cuda")
    model.fused = fused
    model.fold_norm = fold
    return model


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN], ids=["plain", "llama3", "yarn"])
@pytest.mark.parametrize("batch,fold", [(5, False), (2, True), (1, False)])
def test_fused_rows_that_share_a_prompt(batch, fold, scaling):
    """The kernels against the plain route, sharing; and against rows with copies of the prompt."""
    cfg = config(scaling)
    whole = du.whole_model(cfg)
    tokens = answers(cfg, batch, 3, "cuda")
    fused = gpu_model(cfg, whole, fold=fold)
    got = shared_steps(fused, cfg, PROMPT, tokens, "cuda")
    close(got, shared_steps(gpu_model(cfg, whole, fused=False), cfg, PROMPT, tokens, "cuda"))
    close(got, copied_steps(fused, cfg, PROMPT, tokens, "cuda"))


@pytest.mark.gpu
def test_a_captured_step_is_replayed_on_another_prompt():
    """The step is captured once; then another, longer prompt is stepped into the same cache and
    shared, and the replay gives what an eager step gives."""
    cfg = config(LLAMA3)
    model = gpu_model(cfg)
    batch, room = 4, 3
    tokens, positions = torch.zeros(batch, dtype=torch.long, device="cuda"), torch.zeros(batch, dtype=torch.long, device="cuda")
    given = torch.zeros(batch, dtype=torch.long, device="cuda")
    model.allocate_cache(1)
    prefill(model, PROMPT, "cuda")
    model.share_prefix(len(PROMPT), batch, room)
    model.score(tokens, positions, given, top=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.score(tokens, positions, given, top=3)
    for prompt in (PROMPT, PROMPT[::-1] + [90, 3, 3, 17]):
        model.end_prefix()
        prefill(model, prompt, "cuda")
        model.share_prefix(len(prompt), batch, room)
        chosen = answers(cfg, batch, room + 1, "cuda")
        replayed, eager = [], []
        for to in (replayed, eager):
            for t in range(room):
                tokens.copy_(chosen[t]), positions.fill_(t), given.copy_(chosen[t + 1])
                if to is replayed:
                    graph.replay()
                else:
                    out2 = model.score(tokens, positions, given, top=3)
                to.append([x.clone() for x in (out if to is replayed else out2)])
        for a, b in zip(replayed, eager):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    del graph, out
    from linnet_b200 import glue

    glue.decoder_status()


@pytest.mark.gpu
def test_sampled_answers_and_their_log_probabilities():
    """One prompt, six answers: every step takes the alternatives of the last one (row r the r-th most
    probable), and the sums of their log probabilities are those of rows that step through prompt and
    answer by themselves on the plain route.  Six log probabilities of a row, each a logit less the
    logarithm of a sum, are off by twice the logits' tolerance each."""
    cfg = config(YARN)
    whole = du.whole_model(cfg)
    model = gpu_model(cfg, whole)
    batch, steps, rows = 6, 6, torch.arange(6, device="cuda")
    model.allocate_cache(1)
    prefill(model, PROMPT[:-1], "cuda")
    none = torch.full((1,), -1, device="cuda")
    first = model.score(torch.tensor(PROMPT[-1:], device="cuda"), torch.tensor([len(PROMPT) - 1], device="cuda"), none, top=batch)
    model.share_prefix(len(PROMPT), batch, steps)
    chosen, total = [first.top_tokens[0].clone()], first.top_logprobs[0].clone()
    for t in range(steps - 1):
        at = torch.full((batch,), t, device="cuda")
        options = model.score(chosen[-1], at, torch.full((batch,), -1, device="cuda"), top=batch)
        assert torch.equal(options.logprob, torch.zeros_like(options.logprob))
        assert (options.top_logprobs[:, :-1] >= options.top_logprobs[:, 1:]).all() and (options.entropy > 0).all()
        following = options.top_tokens[rows, rows]
        # the step again, now with the token that was chosen: the same numbers, and the cache as it was
        again = model.score(chosen[-1], at, following, top=0)
        assert torch.equal(again.logprob, options.top_logprobs[rows, rows]) and torch.equal(again.entropy, options.entropy)
        chosen.append(following)
        total = total + again.logprob
    plain = gpu_model(cfg, whole, fused=False)
    plain.allocate_cache(batch)
    want, largest = torch.zeros(batch, device="cuda", dtype=torch.double), 0.0
    sequence = [torch.full((batch,), p, device="cuda") for p in PROMPT] + chosen
    for at, token in enumerate(sequence[:-1]):
        logits = plain.step(token, torch.full((batch,), at, device="cuda")).double()
        if at >= len(PROMPT) - 1:
            want += torch.log_softmax(logits, dim=-1)[rows, sequence[at + 1]]
            largest = max(largest, logits.abs().max().item())
    assert (total.double() - want).abs().max().item() <= steps * 2 * 2 * 3e-2 * largest
