"""Rotary positions, shared-prefix attention and token log probabilities where an offset in numbers
passes 2^31 (and 2^32 in bytes): what lies there has to come out as it does from a tensor of its own."""

from __future__ import annotations

import pytest
import torch

from linnet_b200 import _lib, glue

pytestmark = pytest.mark.gpu
FAR = (1 << 31) + (1 << 20)  # numbers


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    torch.cuda.empty_cache()
    _lib.check(_lib.load().b200q_int4_gemm_status())
    glue.decoder_status()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_of_rows_far_apart(layout):
    """Two tokens 2^31 numbers apart in memory, in place and not."""
    room = torch.zeros(FAR + 4096, device="cuda", dtype=torch.bfloat16)
    q = room.as_strided((2, 4, 64), (FAR, 64, 1))
    k = room.as_strided((2, 2, 64), (FAR, 64, 1), 1024)
    q.copy_(torch.randn(2, 4, 64, device="cuda")), k.copy_(torch.randn(2, 2, 64, device="cuda"))
    positions = torch.tensor([5, 70000], device="cuda")
    frequencies, _ = glue.rope_frequencies(64, 1e4)
    want = glue.rotary(q.contiguous(), k.contiguous(), positions, frequencies, layout=layout)
    got = glue.rotary(q, k, positions, frequencies, layout=layout)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    glue.rotary(q, k, positions, frequencies, layout=layout, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_slots_and_keys_far_into_a_cache():
    """A cache of 2^25 slots of 64 numbers: written at its end, attended there, against a short cache."""
    slots = FAR // 64
    cache = torch.zeros(2, 1, 1, slots, 64, device="cuda", dtype=torch.bfloat16)
    short = torch.zeros(2, 1, 1, 130, 64, device="cuda", dtype=torch.bfloat16)
    qkv = torch.randn(1, 3 * 64, device="cuda").to(torch.bfloat16)
    frequencies, _ = glue.rope_frequencies(64, 1e4)
    at = slots - 2
    q = glue.rotary_cache(qkv, torch.tensor([at], device="cuda"), frequencies, cache[0], cache[1], 1, 1)
    other = glue.rotary_cache(qkv, torch.tensor([1], device="cuda"), frequencies, short[0], short[1], 1, 1, offset=at - 1)
    assert torch.equal(q, other) and torch.equal(cache[:, 0, 0, at], short[:, 0, 0, 1])
    assert int((cache != 0).any(dim=-1).sum()) == 2
    # as a prefix whose first key is far from the beginning: its last 129 positions
    end = torch.randn(2, 1, 129, 64, device="cuda").to(torch.bfloat16)
    cache[:, 0, :, -129:] = end
    none = torch.zeros(1, 1, 0, 64, device="cuda", dtype=torch.bfloat16)
    row = torch.tensor([-1], device="cuda")
    far = glue.prefix_attention(q, cache[0, 0, :, -129:], cache[1, 0, :, -129:], none, none, row)
    assert torch.equal(far, glue.prefix_attention(q, end[0], end[1], none, none, row))
    # and all of it, where one key far in has all the weight (its score is 2^7 above the others', which are 0)
    cache.zero_()
    cache[0, 0, 0, at, 0], cache[1, 0, 0, at] = 128.0, 3.0
    q = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1.0
    whole = glue.prefix_attention(q, cache[0, 0], cache[1, 0], none, none, row, scale=1.0)
    assert torch.equal(whole, torch.full_like(whole, 3.0))  # e^-128 * 2^25 is nothing beside 1
    own = torch.tensor([at], device="cuda")
    nothing = cache[0, 0, :, :0]
    assert torch.equal(glue.prefix_attention(q, nothing, nothing, cache[0], cache[1], own, scale=1.0), whole)
    # up to the slot before it: equal weights of zeros
    assert not glue.prefix_attention(q, nothing, nothing, cache[0], cache[1], own - 1, scale=1.0).any()


def test_logits_far_into_a_tensor():
    vocab = 100_000
    rows = FAR // vocab + 1
    logits = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    logits[-3:] = torch.randn(3, vocab, device="cuda")
    tokens = torch.full((rows,), 7, device="cuda")
    got, last = glue.token_logprobs(logits, tokens, 4), glue.token_logprobs(logits[-3:].clone(), tokens[-3:].clone(), 4)
    # (other rows a block: sums in another order, so not the same bits; 2^-15 is the bound of the other tests for 10^5 logits)
    for mine, want in zip(got, last):
        torch.testing.assert_close(mine[-3:], want, rtol=2.0 ** -15, atol=2.0 ** -15)
    assert torch.equal(got.top_tokens[0].cpu(), torch.arange(4))  # equal ones: the lower index first
