"""A shared prompt of many positions: the answers' rotary positions go with those that the prompt's keys
were turned by when it was stepped.

Without scaling the prompt's angles are formed in f32: position times frequency is off by half a step,
2^-24 of the angle, and a cosine or sine by 2^-23.  The answers' angles are formed in f64, of the same
frequencies, and their cosine and sine rounded to f32, 2^-24.  So a number of a pair (a, b) may differ
by (angle * 2^-24 + 2^-22) (|a| + |b|) between the two, f32 products included.  Frequencies that differ
by a step of f32 would add angle * 2^-23."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from linnet_b200 import decoder as dec
from linnet_b200.rope import RopeScaling, frequencies
from tests import decoder_util as du

FAR = 1 << 17


def far_model(linear, device="cpu", scaling=None) -> dec.Int4Decoder:
    cfg = dataclasses.replace(dec.DecoderConfig.tiny(), max_seq=FAR, rope_theta=500000.0, rope_scaling=scaling)
    model = du.rank_model(cfg, du.whole_model(cfg), 0, 1, linear, device=device)
    model.fused = device != "cpu"
    model.allocate_cache(1)
    return model


def allowed(positions: torch.Tensor, freqs: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    size = (x[..., :half].abs() + x[..., half:].abs()).double()
    angle = positions.double()[:, None] * freqs.double()
    return (size * (angle * 2.0 ** -24 + 2.0 ** -22)[:, None]).repeat(1, 1, 2)


def test_answers_turn_by_the_frequencies_of_the_prompt():
    model = far_model(du.oracle_linear)
    model.share_prefix(FAR, 1, 1)
    gen = torch.Generator().manual_seed(3)
    positions = torch.cat([torch.arange(64), torch.randint(64, 1 << 24, (4000,), generator=gen), torch.tensor([FAR - 1, (1 << 24) - 1])])
    x = torch.randn(len(positions), 2, model.cfg.head_dim, generator=gen)
    prompt = dec.rotary(x, positions, model.cfg.rope_theta).double()
    answer = dec.rotary_by(x, positions, model.frequencies, model.rope_factor).double()
    assert bool(((prompt - answer).abs() <= allowed(positions, model.frequencies, x)).all())


def test_scaled_frequencies_are_exact():
    """With a scaling both the prompt and the answers are turned by the f64 numbers."""
    scaling = RopeScaling("llama3", 8.0)
    model = far_model(du.oracle_linear, scaling=scaling)
    numbers, _ = frequencies(model.cfg.head_dim, 500000.0, scaling)
    model.share_prefix(FAR, 1, 1)
    assert model.frequencies.tolist() == numbers


@pytest.mark.gpu
def test_answers_turn_by_the_frequencies_of_the_table():
    """The table holds cosine and sine of fl32(position * frequency): with the answers' frequencies that
    product is computed here, in f32, and the table is within two steps of its cosine and sine."""
    from linnet_b200 import kernels

    model = far_model(kernels.int4_linear, "cuda")
    model.share_prefix(FAR - 2, 2, 2)
    single = model.frequencies.float()
    assert torch.equal(single.double(), model.frequencies)
    angle = (torch.arange(FAR, device="cuda", dtype=torch.float32)[:, None] * single).double()
    table = model.rope_table.double()
    assert (table[..., 0] - angle.cos()).abs().max().item() <= 2.0 ** -22
    assert (table[..., 1] - angle.sin()).abs().max().item() <= 2.0 ** -22


@pytest.mark.gpu
def test_keys_of_far_positions():
    """A token's key in the first layer, written by the step of the prompt and by that of an answer at the
    same position; each of them is rounded to bf16 once more, 2^-8 of itself."""
    from linnet_b200 import kernels

    model = far_model(kernels.int4_linear, "cuda")
    token, zero = torch.tensor([7], device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
    model.step(token, zero)
    x = model.cache_k[0][0, :, 0].float()[None]  # as it is before it is turned: at position 0 it stays
    for at in (1000, 65537, FAR - 1):
        position = torch.tensor([at], device="cuda")
        model.step(token, position)
        prompt = model.cache_k[0][0, :, at].double()
        model.share_prefix(at, 1, 1)
        model.step(token, zero)
        answer = model.cache_k[0][0, :, 0].double()
        bound = allowed(position, model.frequencies, x)[0] + 2.0 ** -8 * (prompt.abs() + answer.abs())
        assert bool(((prompt - answer).abs() <= bound).all()), at
        model.end_prefix()
