"""Calls of the operators for many answers to one prompt that are refused before anything is allocated or
launched."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from linnet_b200 import _lib, glue


@pytest.mark.gpu
@pytest.mark.parametrize("top", [-1, 33, 1 << 45, 8])
def test_alternatives_that_there_are_none_of(top):
    """An absurd number is no question of memory; more than the row has are refused too."""
    logits = torch.zeros(2, 7 if top == 8 else 1000, device="cuda")
    tokens = torch.zeros(2, dtype=torch.long, device="cuda")
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    with pytest.raises(ValueError, match="alternatives of a row"):
        glue.token_logprobs(logits, tokens, top)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


def _rotary_status(tokens, nq, nkv, head_dim, q_out, k_out) -> str:
    """What `b200q_rotary` says of outputs of these strides (of tokens and heads)."""
    lib, memory = _lib.load(), torch.zeros(64, dtype=torch.float64)
    at = memory.data_ptr()
    dense = (nq * head_dim, head_dim, nkv * head_dim, head_dim)
    status = lib.b200q_rotary(at, at, at, at, at, at, tokens, nq, nkv, head_dim, 1, *dense, *q_out, *k_out, 1.0, 0, 1, None)
    return _lib.last_error() if status else ""


@pytest.mark.skipif(torch.cuda.is_available(), reason="host memory: only where no kernel can be launched")
@pytest.mark.parametrize("tokens,nq,nkv,head_dim,q_out,k_out,wrong", [
    (3, 2, 1, 64, (0, 64), (64, 64), True),           # the same memory for every token
    (3, 2, 1, 64, (128, 0), (64, 64), True),          # for every head
    (3, 2, 1, 64, (64, 64), (64, 64), True),          # a token's second head is the next one's first
    (3, 2, 1, 64, (127, 64), (64, 64), True),
    (3, 2, 1, 64, (64, 191), (64, 64), True),         # [heads, tokens, D], a number short
    (3, 2, 2, 64, (128, 64), (128, 32), True),        # keys
    (3, 2, 1, 64, (128, 64), (63, 64), True),
    (3, 1, 1, 64, (-32, 0), (64, 64), True),
    (3, 2, 1, 64, (64, 192), (64, 64), False),        # [heads, tokens, D]
    (3, 2, 1, 64, (-128, 64), (-64, 64), False),
    (1, 2, 1, 64, (0, 64), (0, 0), False),            # of one token or head the stride is not read
    (3, 1, 1, 64, (64, 0), (64, 0), False),
    (1, 1, 1, 64, (0, 0), (0, 0), False),
    (3, 2, 1, 64, (1 << 62, 64), (64, 1 << 62), False)])
def test_rotary_outputs_that_overlap_themselves(tokens, nq, nkv, head_dim, q_out, k_out, wrong):
    """What is taken goes on to the launch, which fails here for want of a GPU."""
    said = _rotary_status(tokens, nq, nkv, head_dim, q_out, k_out)
    assert said and ("overlaps itself" in said) == wrong, said


@pytest.mark.gpu
def test_rotary_refuses_an_expanded_output():
    q = torch.randn(4, 6, 64, device="cuda", dtype=torch.bfloat16)
    positions, freq = torch.arange(4, device="cuda"), torch.ones(32, device="cuda", dtype=torch.float64)
    want, _ = glue.rotary(q, None, positions, freq)
    for out in (torch.empty_like(q[:1]).expand(4, 6, 64), torch.empty_like(q[:, :1]).expand(4, 6, 64)):
        with pytest.raises(ValueError, match="overlaps itself"):
            glue.rotary(q, None, positions, freq, out=(out, None))
        with pytest.raises(ValueError, match="overlaps itself"):
            glue.rotary(q, q, positions, freq, out=(torch.empty_like(q), out))
    by_head = torch.empty(6, 4, 64, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    wide = torch.empty(4, 20, 72, device="cuda", dtype=torch.bfloat16)[:, 3:9, :64]
    for out in (by_head, wide, q):
        got, _ = glue.rotary(q.clone() if out is not q else q, None, positions, freq, out=(out, None))
        assert got is out and torch.equal(out, want)


def _dual(t: torch.Tensor) -> torch.Tensor:
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rotary", "rotary_cache", "prefix_attention", "token_logprobs"])
def test_tangents_are_refused(which):
    """In forward mode too there is no derivative, and none is dropped: an input with a tangent is refused,
    under torch.no_grad as well (which leaves forward mode on); one without passes."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).bfloat16()  # noqa: E731
    freq, at = torch.ones(32, device="cuda", dtype=torch.float64), torch.zeros(3, device="cuda", dtype=torch.long)
    calls = {
        "rotary": (lambda q, k: glue.rotary(q, k, at, freq), [make(3, 4, 64), make(3, 2, 64)]),
        "rotary_cache": (lambda x, k, v: glue.rotary_cache(x, at, freq, k, v, 4, 2), [make(3, 8 * 64), make(3, 2, 5, 64), make(3, 2, 5, 64)]),
        "prefix_attention": (lambda q, a, b, c, d: glue.prefix_attention(q, a, b, c, d, at),
                             [make(3, 4, 64), make(2, 9, 64), make(2, 9, 64), make(3, 2, 5, 64), make(3, 2, 5, 64)]),
        "token_logprobs": (lambda x: glue.token_logprobs(x, at), [make(3, 100)])}
    call, inputs = calls[which]
    with forward_ad.dual_level():
        call(*inputs)
        for i in range(len(inputs)):
            with pytest.raises(RuntimeError, match="no derivative"):
                call(*[_dual(t) if j == i else t for j, t in enumerate(inputs)])
            with torch.no_grad(), pytest.raises(RuntimeError, match="no derivative"):
                call(*[_dual(t) if j == i else t for j, t in enumerate(inputs)])
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.func.jvp(call, tuple(inputs), tuple(torch.ones_like(t) for t in inputs))
    call(*inputs)


@pytest.mark.gpu
def test_frequencies_that_ask_for_a_derivative_are_refused():
    q, at = torch.randn(3, 4, 64, device="cuda").bfloat16(), torch.zeros(3, device="cuda", dtype=torch.long)
    qkv, cache = torch.randn(3, 8 * 64, device="cuda").bfloat16(), torch.zeros(2, 3, 2, 5, 64, device="cuda", dtype=torch.bfloat16)
    freq = torch.ones(32, device="cuda", dtype=torch.float64)
    calls = (lambda f: glue.rotary(q, None, at, f), lambda f: glue.rotary_cache(qkv, at, f, cache[0], cache[1], 4, 2),
             lambda f: glue.rotary_table(9, f))
    for call in calls:
        with pytest.raises(RuntimeError, match="no derivative"):
            call(freq.clone().requires_grad_())
        with torch.no_grad():
            call(freq.clone().requires_grad_())
        with forward_ad.dual_level():
            call(freq)
            with pytest.raises(RuntimeError, match="no derivative"):
                call(_dual(freq))
