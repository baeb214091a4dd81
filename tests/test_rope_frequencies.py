"""`linnet_b200.rope`: the frequencies against their definitions written out, and what is refused; the
refusals of the entry points that need no GPU."""

from __future__ import annotations

import math

import pytest
import torch

from linnet_b200 import glue, rope


@pytest.mark.parametrize("rotary", [2, 48, 64, 128])
def test_unscaled_and_linear_and_ntk(rotary):
    plain, factor = rope.frequencies(rotary, 10000.0)
    assert factor == 1.0 and plain[0] == 1.0 and len(plain) == rotary // 2
    for i, f in enumerate(plain):
        assert f == pytest.approx(math.exp(-math.log(10000.0) * 2 * i / rotary), rel=1e-14)
    linear, factor = rope.frequencies(rotary, 10000.0, rope.RopeScaling("linear", 4.0))
    assert factor == 1.0 and linear == [f / 4.0 for f in plain]
    ntk, factor = rope.frequencies(rotary, 10000.0, rope.RopeScaling("ntk", 4.0))
    assert factor == 1.0 and ntk[0] == 1.0
    if rotary > 2:  # the last pair turns exactly `factor` times slower
        assert ntk[-1] == pytest.approx(plain[-1] / 4.0, rel=1e-12)


def test_llama3_bands():
    plain, _ = rope.frequencies(128, 500000.0)
    scaled, factor = rope.frequencies(128, 500000.0, rope.RopeScaling("llama3", 8.0, 8192, low=1.0, high=4.0))
    assert factor == 1.0
    for f, g in zip(plain, scaled):
        wavelength = 2 * math.pi / f
        if wavelength < 8192 / 4:
            assert g == f
        elif wavelength > 8192:
            assert g == pytest.approx(f / 8, rel=1e-14)
        else:
            smooth = (8192 / wavelength - 1) / 3
            assert g == pytest.approx((1 - smooth) * f / 8 + smooth * f, rel=1e-12)
    assert any(f / 8 < g < f for f, g in zip(plain, scaled))


def test_yarn_ramp_and_factor():
    plain, _ = rope.frequencies(64, 10000.0)
    scaled, factor = rope.frequencies(64, 10000.0, rope.RopeScaling("yarn", 16.0, 4096))
    assert factor == pytest.approx(0.1 * math.log(16.0) + 1.0, rel=1e-15)
    ratios = [g / f for f, g in zip(plain, scaled)]
    assert ratios[0] == 1.0 and ratios[-1] == pytest.approx(1 / 16, rel=1e-12)
    assert all(a >= b for a, b in zip(ratios, ratios[1:]))
    _, given = rope.frequencies(64, 10000.0, rope.RopeScaling("yarn", 16.0, 4096, attention_factor=1.0))
    assert given == 1.0


@pytest.mark.parametrize("kwargs", [
    {"kind": "dynamic", "factor": 2.0}, {"kind": "linear", "factor": 0.5}, {"kind": "linear", "factor": math.nan},
    {"kind": "llama3", "factor": 8.0, "low": 4.0, "high": 1.0}, {"kind": "yarn", "factor": 8.0, "beta_fast": 1.0, "beta_slow": 32.0},
    {"kind": "linear", "factor": 2.0, "original_positions": 0}])
def test_scalings_that_are_refused(kwargs):
    with pytest.raises(ValueError, match="rope scaling"):
        rope.RopeScaling(**kwargs)


def test_frequencies_that_are_refused():
    for rotary, theta in ((0, 1e4), (7, 1e4), (64, 1.0), (64, math.nan)):
        with pytest.raises(ValueError, match="rotary positions"):
            rope.frequencies(rotary, theta)


def test_entries_refuse_tensors_off_the_gpu():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)
    at, freq = torch.zeros(2, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        glue.rotary(x, x, at, freq)
    with pytest.raises(RuntimeError, match="CUDA"):
        glue.rotary_cache(x.view(2, 256), at, freq, cache, cache, 2, 1)
    with pytest.raises(ValueError, match="rotary_table"):
        glue.rotary_table(8, freq)
    with pytest.raises(RuntimeError, match="CUDA"):
        glue.token_logprobs(torch.zeros(2, 8), at)


def test_c_entries_check_shapes_on_the_host():
    from linnet_b200 import _lib

    lib = _lib.load()

    def rotary(tokens=1, nq=1, nkv=0, hd=64, pairs=32, layout=0, dtype=_lib.BF16):
        return lib.b200q_rotary(None, None, None, None, None, None, tokens, nq, nkv, hd, pairs, *([0] * 8), 1.0, layout,
                                dtype, None)

    for bad, message in (({"tokens": -1}, "bad shape"), ({"nq": 0}, "bad shape"), ({"pairs": 33}, "33 pairs"),
                         ({"pairs": 0}, "0 pairs"), ({"hd": 2048, "pairs": 64}, "1024 at most"), ({"layout": 2}, "layout"),
                         ({"dtype": _lib.F32}, "bf16 or f16"), ({}, "null")):
        assert rotary(**bad) == _lib.ERROR and message in _lib.last_error(), bad
    assert rotary(tokens=0) == _lib.OK

    def cache(batch=1, nkv=1, slots=8):
        return lib.b200q_rotary_cache(None, None, None, None, 0, None, None, None, batch, 1, nkv, 64, 32, slots, 1.0, 0,
                                      _lib.F16, None)

    for bad, message in (({"nkv": 0}, "bad shape"), ({"slots": 0}, "bad shape"), ({}, "null")):
        assert cache(**bad) == _lib.ERROR and message in _lib.last_error(), bad
    assert cache(batch=0) == _lib.OK

    def logprobs(rows=1, vocab=8, top=0, dtype=_lib.F32):
        return lib.b200q_token_logprobs(None, None, None, None, None, None, rows, vocab, vocab, top, dtype, None)

    for bad, message in (({"rows": -1}, "rows"), ({"vocab": 0}, "rows"), ({"vocab": (1 << 20) + 1}, "2^20"),
                         ({"top": 33, "vocab": 64}, "0 to 32"), ({"top": 9}, "0 to 8"), ({"top": -1}, "0 to 8"),
                         ({"dtype": 7}, "f32, bf16 or f16"), ({}, "null")):
        assert logprobs(**bad) == _lib.ERROR and message in _lib.last_error(), bad
    assert logprobs(rows=0) == _lib.OK
