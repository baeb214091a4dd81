"""`glue.rotary`, `rotary_cache` and `rotary_table` against rotations in 64 bits.

What may differ: the result's own rounding (half a step of its type), and of cosine and sine in f32
their rounding, that of the angle's remainder (2^-24 of at most pi) and of the two products and
their sum: below 2^-20 of the pair's numbers, times the factor.  The angle itself is a product of two
f64: the one formed here is off by half a step, 2^-53 of itself; the kernel's by three of those
(1 / 2 pi, the frequency in turns, the product), so at position 2^40 by 4 * 2^-53 * 2^40 = 2^-11 of a
radian: that times the pair's numbers."""

from __future__ import annotations

import pytest
import torch

from linnet_b200 import glue, rope

pytestmark = pytest.mark.gpu


def _turned(x, positions, freq, layout, factor):
    """(results, allowances) in f64."""
    pairs = freq.numel()
    angle = positions.double()[:, None] * freq[None]
    cos, sin = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]
    y, slack = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    at = torch.arange(pairs, device=x.device)
    first, second = (at, at + pairs) if layout == "half" else (2 * at, 2 * at + 1)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    slack[..., first] = slack[..., second] = (a.abs() + b.abs()) * abs(factor) * (2.0 ** -20 + angle.abs()[:, None] * 2.0 ** -51)
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * half
    return y, slack + y.abs() * half + tiny * (slack > 0)


def _close(got, want, allowed):
    assert got.shape == want.shape
    over = ((got.double() - want).abs() - allowed).max().item() if got.numel() else 0.0
    assert over <= 0.0


def _freq(pairs, dtype=torch.float64):
    return torch.tensor(rope.frequencies(2 * pairs, 500000.0)[0], dtype=dtype, device="cuda")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,nq,nkv,hd,pairs,start,factor", [
    (1, 32, 8, 128, 64, 0, 1.0), (1, 1, 0, 2, 1, 5, 1.0), (7, 3, 1, 64, 32, 1 << 40, 1.0), (2, 4, 2, 80, 20, 3, 1.25),
    (300, 8, 2, 128, 32, 131072, 1.0), (5, 2, 2, 18, 3, 9, 1.0), (33, 28, 4, 128, 56, 10 ** 6, 1.4), (1000, 16, 16, 64, 8, 0, 1.0),
    (3, 1, 1, 1024, 512, 77, 1.0), (2, 5, 1, 72, 32, 0, 1.0)])
def test_rotary(layout, dtype, tokens, nq, nkv, hd, pairs, start, factor):
    gen = torch.Generator(device="cuda").manual_seed(tokens * hd + pairs)
    qkv = torch.randn(tokens, nq + 2 * nkv, hd, device="cuda", generator=gen).to(dtype)
    before = qkv.clone()
    q, k = qkv[:, :nq], qkv[:, nq:nq + nkv] if nkv else None
    positions = start + torch.randperm(tokens, device="cuda", generator=gen)
    freq = _freq(pairs)
    q_out, k_out = glue.rotary(q, k, positions, freq, layout=layout, factor=factor)
    assert q_out.is_contiguous() and torch.equal(qkv, before)
    _close(q_out, *_turned(q, positions, freq, layout, factor))
    if nkv:
        _close(k_out, *_turned(k, positions, freq, layout, factor))
        # in place, inside the projection: the same bits, and v and what is between as they were
        glue.rotary(q, k, positions, freq, layout=layout, factor=factor, out=(q, k))
        assert torch.equal(q, q_out) and torch.equal(k, k_out) and torch.equal(qkv[:, nq + nkv:], before[:, nq + nkv:])
    else:
        assert k_out is None


def test_rotary_of_odd_strides_and_addresses():
    """Rows that begin off 16-byte boundaries take the narrow accesses: the same results."""
    base = torch.randn(9 * 5 * 67 + 1, device="cuda").to(torch.bfloat16)
    odd = base[1:].view(9, 5, 67)[:, :, :64]
    positions, freq = torch.arange(9, device="cuda"), _freq(32)
    got, _ = glue.rotary(odd, None, positions, freq)
    want, _ = glue.rotary(odd.contiguous(), None, positions, freq)
    assert torch.equal(got, want)
    into = torch.full((9 * 5 * 67 + 1,), 7.0, device="cuda", dtype=torch.bfloat16)
    view = into[1:].view(9, 5, 67)[:, :, :64]
    glue.rotary(odd, None, positions, freq, out=(view, None))
    assert torch.equal(view, want) and bool((into[1:].view(9, 5, 67)[:, :, 64:] == 7).all()) and float(into[0]) == 7


def test_rotary_of_nothing_and_of_negative_positions():
    freq = _freq(32)
    empty = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    q, k = glue.rotary(empty, empty, torch.empty(0, dtype=torch.int64, device="cuda"), freq)
    assert q.shape == k.shape == (0, 4, 64)
    x = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    positions = torch.tensor([-1, -70000, 0], device="cuda")
    _close(glue.rotary(x, None, positions, freq)[0], *_turned(x, positions, freq, "half", 1.0))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,nq,nkv,hd,pairs,slots,offset", [
    (1, 32, 8, 128, 64, 64, 0), (3, 4, 2, 64, 16, 5, 1 << 33), (200, 8, 1, 128, 64, 3, 4097), (2, 3, 1, 20, 5, 4, 2),
    (4, 2, 2, 64, 24, 1, 10 ** 6)])
def test_rotary_cache(layout, dtype, batch, nq, nkv, hd, pairs, slots, offset):
    gen = torch.Generator(device="cuda").manual_seed(batch * hd + pairs)
    qkv = torch.randn(batch, (nq + 2 * nkv) * hd, device="cuda", generator=gen).to(dtype)
    cache_k = torch.full((batch, nkv, slots, hd), 7.0, device="cuda", dtype=dtype)
    cache_v = cache_k.clone()
    positions = torch.randint(0, slots, (batch,), device="cuda", generator=gen)
    freq = _freq(pairs)
    q = glue.rotary_cache(qkv, positions, freq, cache_k, cache_v, nq, nkv, layout=layout, factor=1.1, offset=offset)
    heads, rows = qkv.view(batch, nq + 2 * nkv, hd), torch.arange(batch, device="cuda")
    want, allowed = _turned(heads[:, :nq + nkv], positions + offset, freq, layout, 1.1)
    _close(q, want[:, :nq], allowed[:, :nq])
    _close(cache_k[rows, :, positions], want[:, nq:], allowed[:, nq:])
    assert torch.equal(cache_v[rows, :, positions], heads[:, nq + nkv:])
    # every other slot as it was
    cache_k[rows, :, positions] = 7.0
    cache_v[rows, :, positions] = 7.0
    assert bool((cache_k == 7).all()) and bool((cache_v == 7).all())
    # the offset as a word on the device: the same
    again = glue.rotary_cache(qkv, positions, freq, cache_k, cache_v, nq, nkv, layout=layout, factor=1.1,
                              offset=torch.tensor([offset], device="cuda"))
    assert torch.equal(again, q)


def test_rotary_cache_agrees_with_rope_cache():
    """Unscaled, halves, near positions: what the unscaled kernel writes, up to the angles in f32 that it has."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(5, 8 * 64, device="cuda", generator=gen).to(torch.bfloat16)
    caches = [torch.zeros(5, 2, 16, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    positions = torch.arange(5, device="cuda") * 3
    freq = torch.tensor(rope.frequencies(64, 10000.0)[0], dtype=torch.float64, device="cuda")
    a = glue.rotary_cache(qkv, positions, freq, caches[0], caches[1], 4, 2)
    b = glue.rope_cache(qkv, positions, caches[2], caches[3], 4, 2, 10000.0)
    # two roundings to bf16, and angles of at most 12 radians off by 2^-21 of themselves
    for x, y in ((a, b), (caches[0], caches[2])):
        assert bool(((x.float() - y.float()).abs() <= y.float().abs() * 2.0 ** -7 + 8 * 2.0 ** -16).all())
    assert torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("bad", [4, -1, 1 << 40])
def test_a_position_outside_the_cache_is_reported_and_stores_nothing(bad):
    qkv = torch.randn(3, 4 * 64, device="cuda").to(torch.bfloat16)
    around_k = torch.full((5, 1, 4, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    around_v = around_k.clone()
    glue.decoder_status()
    positions = torch.tensor([1, bad, 3], device="cuda")
    glue.rotary_cache(qkv, positions, _freq(32), around_k[1:-1], around_v[1:-1], 2, 1)
    with pytest.raises(ValueError, match="batch row 1"):
        glue.decoder_status()
    for cache in (around_k, around_v):
        assert bool((cache[0] == 7).all()) and bool((cache[2] == 7).all()) and bool((cache[-1] == 7).all())
        assert not bool((cache[1, :, 1] == 7).all()) and not bool((cache[3, :, 3] == 7).all())


def test_rotary_table_is_what_the_fused_kernel_takes():
    freq, factor = glue.rope_frequencies(128, 500000.0, scaling=rope.RopeScaling("yarn", 4.0, 1024))
    table = glue.rotary_table(5000, freq, factor)
    angle = torch.arange(5000, device="cuda").double()[:, None] * freq[None]
    want = torch.stack([angle.cos(), angle.sin()], dim=-1) * factor
    assert table.dtype == torch.float32 and bool(((table.double() - want).abs() <= 2.0 ** -21).all())
    # rope_attention with it: the keys it stores are those of rotary_cache
    gen = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(2, 6 * 128, device="cuda", generator=gen).to(torch.bfloat16)
    caches = [torch.zeros(2, 1, 64, 128, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    positions = torch.tensor([63, 7], device="cuda")
    glue.rope_attention(qkv, positions, table[:64].contiguous(), caches[0], caches[1], 4, 1)
    glue.rotary_cache(qkv, positions, freq, caches[2], caches[3], 4, 1, factor=factor)
    assert bool(((caches[0].float() - caches[2].float()).abs() <= caches[2].float().abs() * 2.0 ** -7 + 2.0 ** -16).all())
    assert torch.equal(caches[1], caches[3])


def test_rotary_in_a_graph_and_on_another_stream():
    x = torch.randn(64, 8, 128, device="cuda").to(torch.bfloat16)
    positions, freq = torch.arange(64, device="cuda"), _freq(64)
    want, _ = glue.rotary(x, None, positions, freq)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other, _ = glue.rotary(x, None, positions, freq)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = glue.rotary(x, None, positions, freq)
    x.mul_(2.0)
    positions.add_(11)
    want, _ = glue.rotary(x, None, positions, freq)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_rotary_refusals():
    x, at, freq = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64, device="cuda"), _freq(32)
    with pytest.raises(RuntimeError, match="types"):
        glue.rotary(x.float(), None, at, freq)
    with pytest.raises(RuntimeError, match="types"):
        glue.rotary(x, x.half(), at, freq)
    with pytest.raises(RuntimeError, match="last dimension"):
        glue.rotary(x.transpose(1, 2), None, at, freq)
    with pytest.raises(RuntimeError, match="no derivative"):
        glue.rotary(x.clone().requires_grad_(), None, at, freq)
    with pytest.raises(ValueError, match="tokens, heads"):
        glue.rotary(x, x[:1], at, freq)
    with pytest.raises(ValueError, match="int64"):
        glue.rotary(x, None, at.int(), freq)
    with pytest.raises(ValueError, match="float64"):
        glue.rotary(x, None, at, freq.float())
    with pytest.raises(ValueError, match="1 to 32"):
        glue.rotary(x, None, at, _freq(33))
    with pytest.raises(ValueError, match="layout"):
        glue.rotary(x, None, at, freq, layout="pairs")
    with pytest.raises(ValueError, match="shapes"):
        glue.rotary(x, None, at, freq, out=(x[:, :2], None))
    cache = torch.zeros(2, 1, 8, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="go together"):
        glue.rotary_cache(x.view(2, 256), at, freq, cache, cache, 3, 1)
    with pytest.raises(RuntimeError, match="contiguous"):
        glue.rotary_cache(x.view(2, 256), at, freq, cache[:, :, :4], cache[:, :, :4], 2, 1)
    with pytest.raises(ValueError, match="offset"):
        glue.rotary_cache(x.view(2, 256), at, freq, cache, cache, 2, 1, offset=torch.zeros(2, dtype=torch.int64, device="cuda"))


def test_keys_of_no_heads_offsets_that_are_no_whole_numbers_and_views_in_place():
    q = torch.randn(3, 4, 64, device="cuda").to(torch.bfloat16)
    positions = torch.arange(3, device="cuda")
    frequencies, _ = glue.rope_frequencies(64, 1e4)
    alone, none = glue.rotary(q, None, positions, frequencies)
    both, empty = glue.rotary(q, q[:, :0], positions, frequencies)
    assert none is None and empty.shape == (3, 0, 64) and torch.equal(alone, both)
    # q and k are views of one projection, turned where they are; v between them stays
    fused = torch.randn(3, 4 + 2 + 2, 64, device="cuda").to(torch.bfloat16)
    before = fused.clone()
    want = glue.rotary(before[:, :4], before[:, 6:], positions, frequencies)
    glue.rotary(fused[:, :4], fused[:, 6:], positions, frequencies, out=(fused[:, :4], fused[:, 6:]))
    assert torch.equal(fused[:, :4], want[0]) and torch.equal(fused[:, 6:], want[1])
    assert torch.equal(fused[:, 4:6], before[:, 4:6])
    cache = torch.zeros(3, 1, 8, 64, device="cuda", dtype=torch.bfloat16)
    qkv = torch.randn(3, 3 * 64, device="cuda").to(torch.bfloat16)
    with pytest.raises(TypeError):
        glue.rotary_cache(qkv, positions, frequencies, cache, cache.clone(), 1, 1, offset=1.5)
