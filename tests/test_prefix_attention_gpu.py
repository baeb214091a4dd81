"""`glue.prefix_attention` against softmax attention in 64 bits.

What may differ, with p the weights of a row (sum 1): each p is rounded to the tensors' type (half a
step, u = eps / 2, of itself), so a result by at most u sum p |v|; the result's own rounding, u of
itself; and in f32 the scores (2^-22 of sum |q k| scale for products and sums, and as much for the
exponential's argument), which move every p by that share of itself: twice that times sum p |v|."""

from __future__ import annotations

import math

import pytest
import torch

from linnet_b200 import _lib, glue

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_expired():
    yield
    _lib.check(_lib.load().b200q_int4_gemm_status())


def _want(q, pk, pv, ck, cv, positions, scale=None, length=None):
    """(results, allowances) [B, nq * D] in f64; row by row."""
    batch, nq, hd = q.shape
    nkv = pk.shape[0]
    rep, scale = nq // nkv, hd ** -0.5 if scale is None else scale
    out = torch.zeros(batch, nq, hd, dtype=torch.float64, device=q.device)
    allowed = torch.zeros_like(out)
    u = torch.finfo(q.dtype).eps / 2
    length = pk.shape[1] if length is None else length
    for b, last in enumerate(positions.tolist()):
        k = torch.cat([pk[:, :length], ck[b, :, :last + 1]], dim=1).double()
        v = torch.cat([pv[:, :length], cv[b, :, :last + 1]], dim=1).double()
        if k.shape[1] == 0:
            continue
        x = q[b].double().view(nkv, rep, hd)
        p = torch.softmax(x @ k.transpose(1, 2) * scale, dim=-1)
        size = (x.abs() @ k.abs().transpose(1, 2)).amax(dim=-1, keepdim=True) * abs(scale)
        y = p @ v
        out[b] = y.reshape(nq, hd)
        allowed[b] = (u * y.abs() + (u + 2 * size * 2.0 ** -21 + 2.0 ** -18) * (p @ v.abs())).reshape(nq, hd)
    tiny = torch.finfo(q.dtype).smallest_normal * u * 2
    return out.flatten(1), allowed.flatten(1) + tiny


def _inputs(batch, nq, nkv, hd, prefix, slots, dtype, seed=0, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + batch * 31 + prefix)
    make = lambda *shape, std=1.0: (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)  # noqa: E731
    q, pk, pv = make(batch, nq, hd, std=spread), make(nkv, prefix, hd), make(nkv, prefix, hd)
    ck, cv = make(batch, nkv, slots, hd), make(batch, nkv, slots, hd)
    positions = torch.randint(-1, slots, (batch,), device="cuda", generator=gen) if slots else torch.full((batch,), -1, device="cuda")
    return q, pk, pv, ck, cv, positions


def _check(q, pk, pv, ck, cv, positions, **kwargs):
    got = glue.prefix_attention(q, pk, pv, ck, cv, positions, **kwargs)
    want, allowed = _want(q, pk, pv, ck, cv, positions, kwargs.get("scale"))
    assert got.shape == want.shape and got.dtype == q.dtype
    over = ((got.double() - want).abs() / allowed).max().item()
    assert over <= 1.0, over
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,nq,nkv,hd,prefix,slots", [
    (1, 1, 1, 64, 1, 1), (1, 4, 1, 128, 128, 1), (2, 4, 2, 64, 100, 5), (3, 8, 2, 128, 129, 128), (5, 14, 2, 64, 1000, 130),
    (33, 32, 8, 128, 300, 7), (64, 8, 2, 128, 2000, 257), (65, 8, 4, 64, 511, 31), (127, 6, 2, 128, 640, 3), (300, 4, 2, 64, 130, 40),
    (16, 16, 1, 128, 4097, 0), (4, 128, 1, 128, 700, 9), (3, 64, 1, 64, 257, 300), (40, 7, 1, 128, 900, 64), (9, 10, 2, 128, 0, 500),
    (200, 8, 8, 128, 384, 129), (1, 32, 8, 128, 10000, 1000), (700, 4, 4, 64, 64, 2)])
def test_prefix_attention(dtype, batch, nq, nkv, hd, prefix, slots):
    _check(*_inputs(batch, nq, nkv, hd, prefix, slots, dtype))


@pytest.mark.parametrize("hd", [64, 128])
def test_peaked_scores_move_the_maximum(hd):
    """Scores that rise along the keys by hundreds: the running maximum moves, O and l are rescaled."""
    q, pk, pv, ck, cv, positions = _inputs(70, 8, 2, hd, 3000, 200, torch.bfloat16, spread=8.0)
    ramp = torch.linspace(0.1, 4.0, 3000, device="cuda")[:, None]
    _check(q, (pk.float() * ramp).to(pk.dtype), pv, ck, cv, positions)
    _check(q, (pk.float() * ramp.flip(0)).to(pk.dtype), pv, ck, cv, positions)


def test_rows_without_keys_and_scale():
    q, pk, pv, ck, cv, positions = _inputs(20, 8, 2, 128, 0, 100, torch.bfloat16)
    positions[3] = positions[11] = -1
    got = _check(q, pk, pv, ck, cv, positions, scale=0.3)
    assert bool((got[3] == 0).all()) and bool((got[11] == 0).all())
    positions.fill_(-1)
    assert bool((glue.prefix_attention(q, pk, pv, ck, cv, positions) == 0).all())
    q, pk, pv, ck, cv, positions = _inputs(20, 8, 2, 128, 77, 100, torch.bfloat16)
    _check(q, pk, pv, ck, cv, positions.fill_(-1), scale=1e-30)  # even weights
    for scale in (0.0, -0.1, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            glue.prefix_attention(q, pk, pv, ck, cv, positions, scale=scale)
    empty = glue.prefix_attention(q[:0], pk, pv, ck[:0], cv[:0], positions[:0])
    assert empty.shape == (0, 8 * 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
def test_nothing_behind_the_last_key_is_read_into_the_result(dtype, hd):
    q, pk, pv, ck, cv, positions = _inputs(37, 6, 2, hd, 300, 200, dtype)
    want = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    for fill in (math.nan, math.inf, -math.inf):
        room = torch.full((2, 2, 512, hd), fill, device="cuda", dtype=dtype)
        room[0, :, :300], room[1, :, :300] = pk, pv
        k, v = ck.clone(), cv.clone()
        behind = torch.arange(200, device="cuda")[None] > positions[:, None]
        k.masked_fill_(behind[:, None, :, None], fill)
        v.masked_fill_(behind[:, None, :, None], fill)
        assert torch.equal(glue.prefix_attention(q, room[0][:, :300], room[1][:, :300], k, v, positions), want)
        # the same with the prefix's length on the device, over the whole room
        length = torch.tensor([300], device="cuda")
        got = glue.prefix_attention(q, room[0], room[1], k, v, positions, prefix_length=length)
        expected, allowed = _want(q, pk, pv, ck, cv, positions)
        assert bool(((got.double() - expected).abs() <= allowed).all())


def test_prefix_length_on_the_device_in_a_graph():
    q, pk, pv, ck, cv, positions = _inputs(24, 8, 2, 128, 1500, 64, torch.bfloat16)
    length = torch.tensor([1500], device="cuda")
    graph = torch.cuda.CUDAGraph()
    glue.prefix_attention(q, pk, pv, ck, cv, positions, prefix_length=length)
    with torch.cuda.graph(graph):
        got = glue.prefix_attention(q, pk, pv, ck, cv, positions, prefix_length=length)
    for n, moved in ((1500, 0), (1, 3), (0, 1), (1377, 0), (128, 2)):
        length.fill_(n)
        positions.copy_((positions + moved).clamp(-1, 63))
        graph.replay()
        want, allowed = _want(q, pk, pv, ck, cv, positions, length=n)
        assert bool(((got.double() - want).abs() <= allowed).all()), n
    glue.decoder_status()
    for n, same in ((-5, 0), (1 << 40, 1500)):
        length.fill_(n)
        graph.replay()
        want, allowed = _want(q, pk, pv, ck, cv, positions, length=same)
        assert bool(((got.double() - want).abs() <= allowed).all())
        with pytest.raises(ValueError, match="batch row 0"):
            glue.decoder_status()


@pytest.mark.parametrize("bad", [-2, 64, 1 << 40])
def test_a_position_outside_the_cache_counts_as_none_and_is_reported(bad):
    q, pk, pv, ck, cv, positions = _inputs(10, 8, 2, 128, 200, 64, torch.bfloat16)
    positions[6] = -1
    want = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    glue.decoder_status()
    positions[6] = bad
    got = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    with pytest.raises(ValueError, match="batch row 6"):
        glue.decoder_status()
    assert torch.equal(got, want)


def test_strides():
    """Queries as a view of the projection, prefix and caches as parts of longer ones and of other layouts."""
    q, pk, pv, ck, cv, positions = _inputs(21, 12, 4, 64, 333, 50, torch.float16)
    want = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    wide = torch.randn(21, 12 + 8, 64, device="cuda").half()
    wide[:, :12] = q
    by_key = pk.transpose(0, 1).contiguous().transpose(0, 1)          # [P, nkv, D] in memory
    both = torch.full((21, 50, 2, 4, 64 + 8), 3.0, device="cuda", dtype=torch.float16)  # [B, S, K|V, nkv, D and some]
    both[:, :, 0, :, :64], both[:, :, 1, :, :64] = ck.transpose(1, 2), cv.transpose(1, 2)
    got = glue.prefix_attention(wide[:, :12], by_key, pv, both[:, :, 0, :, :64].transpose(1, 2), both[:, :, 1, :, :64].transpose(1, 2), positions)
    assert torch.equal(got, want)
    one = glue.prefix_attention(q, pk, pv, ck[:, :, :1], cv[:, :, :1], positions.clamp(max=0))
    alone, allowed = _want(q, pk, pv, ck, cv, positions.clamp(max=0))
    assert bool(((one.double() - alone).abs() <= allowed).all())


def test_agrees_with_decode_attention():
    """No prefix: what the framework's attention over one cache a row gives, up to roundings."""
    q, pk, pv, ck, cv, positions = _inputs(12, 8, 2, 128, 0, 300, torch.bfloat16)
    positions.clamp_(min=0)
    a = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    b = glue.decode_attention(q, ck, cv, positions)
    _, allowed = _want(q, pk, pv, ck, cv, positions)
    assert bool(((a.double() - b.double()).abs() <= 2 * allowed).all())


def test_the_same_bits_every_time_on_any_stream_and_two_at_once():
    q, pk, pv, ck, cv, positions = _inputs(50, 8, 2, 128, 1111, 90, torch.bfloat16)
    other = _inputs(30, 4, 1, 64, 700, 40, torch.float16)
    want, want_other = glue.prefix_attention(q, pk, pv, ck, cv, positions), glue.prefix_attention(*other)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, args in zip(streams, ((q, pk, pv, ck, cv, positions), other)):
            with torch.cuda.stream(stream):
                got.append(glue.prefix_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got[0::2]) and all(torch.equal(x, want_other) for x in got[1::2])


def test_nan_and_infinity_among_the_keys_show():
    q, pk, pv, ck, cv, positions = _inputs(6, 4, 2, 64, 150, 40, torch.bfloat16)
    positions.fill_(39)
    ck[2, 1, 5] = math.nan
    cv[4, 0, 7] = math.inf
    got = glue.prefix_attention(q, pk, pv, ck, cv, positions).view(6, 4, 64)
    assert bool(got[2, 2:].isnan().all()) and bool((got[4, :2] == math.inf).all())
    rest = torch.ones(6, 4, dtype=torch.bool, device="cuda")
    rest[2, 2:] = rest[4, :2] = False
    assert bool(torch.isfinite(got[rest]).all())


def test_refusals():
    q, pk, pv, ck, cv, positions = _inputs(4, 8, 2, 64, 100, 20, torch.bfloat16)
    bad = [
        (RuntimeError, "types", (q.float(), pk, pv, ck, cv, positions)),
        (RuntimeError, "types", (q, pk.half(), pv.half(), ck, cv, positions)),
        (RuntimeError, "last dimension", (q, pk.transpose(1, 2), pv, ck, cv, positions)),
        (RuntimeError, "no derivative", (q.clone().requires_grad_(), pk, pv, ck, cv, positions)),
        (ValueError, "go together", (q, pk[:1], pv[:1], ck, cv, positions)),
        (ValueError, "go together", (q[:3], pk, pv, ck, cv, positions)),
        (ValueError, "go together", (q, pk, pv[:, :50], ck, cv, positions)),
        (ValueError, "int64", (q, pk, pv, ck, cv, positions.int())),
        (ValueError, "whole number", (q[:, :7], pk, pv, ck, cv, positions)),
        (ValueError, "64 or 128", (q[..., :32], pk[..., :32], pv[..., :32], ck[..., :32], cv[..., :32], positions)),
        (ValueError, "16-byte steps", (torch.zeros(4, 8, 65, device="cuda", dtype=torch.bfloat16)[..., :64], pk, pv, ck, cv, positions)),
    ]
    for error, message, args in bad:
        with pytest.raises(error, match=message):
            glue.prefix_attention(*args)
    for length in (3, torch.tensor([3]), torch.tensor([3], device="cuda", dtype=torch.int32)):
        with pytest.raises(ValueError, match="prefix_length"):
            glue.prefix_attention(q, pk, pv, ck, cv, positions, prefix_length=length)
    odd = torch.zeros(2 * 100 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 100, 64)
    with pytest.raises(ValueError, match="16-byte aligned"):
        glue.prefix_attention(q, odd, pv, ck, cv, positions)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,slots", [(200, 5), (1000, 0), (0, 300)])
def test_scores_of_minus_infinity_have_no_weight(dtype, prefix, slots):
    """Keys that score -inf for every row fill the first tiles; the others count as if those were not there."""
    q, pk, pv, ck, cv, positions = _inputs(40, 8, 2, 64, prefix, slots, dtype)
    q[..., 0] = 1.0
    positions.fill_(slots - 1)
    pk[:, :130, 0] = -math.inf
    if prefix == 0:
        ck[:, :, :130, 0] = -math.inf
    got = glue.prefix_attention(q, pk, pv, ck, cv, positions)
    if prefix:
        want, allowed = _want(q, pk[:, 130:], pv[:, 130:], ck, cv, positions)
    else:
        want, allowed = _want(q, pk, pv, ck[:, :, 130:], cv[:, :, 130:], positions - 130)
    assert ((got.double() - want).abs() / allowed).max().item() <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_small_weights_beside_a_large_one(dtype):
    """One key of weight 1 and value 0, 2^20 of 2^-26.5 and value 1: the result is what those come to,
    2^-6.5.  The smallest step of an f16 weight is 2^-24 of 2^-7 of the largest, so each of them is off
    by 2^-32 at most, and all by 2^-12; in bf16 by half a step, u of each.  The result's own rounding
    is u of it again, the f32 sums' and the exponential's share 2^-18 as everywhere."""
    small, count = 2.0 ** -26.5, 2 ** 20
    pk = torch.zeros(1, count + 1, 64, device="cuda", dtype=dtype)
    pv = torch.ones(1, count + 1, 64, device="cuda", dtype=dtype)
    pk[0, 5, 0], pv[0, 5] = 1.0, 0.0
    q = torch.zeros(3, 1, 64, device="cuda", dtype=dtype)
    q[..., 0] = 8.0
    empty = torch.zeros(3, 1, 0, 64, device="cuda", dtype=dtype)
    # score 8 * scale of the large one: ln 2^26.5, whatever the product's rounding
    got = glue.prefix_attention(q, pk, pv, empty, empty, torch.full((3,), -1, device="cuda"), scale=26.5 * math.log(2) / 8)
    want = count * small / (1 + count * small)
    u = torch.finfo(dtype).eps / 2
    each = 2.0 ** -32 if dtype == torch.float16 else u * small
    assert (got.double() - want).abs().max().item() <= count * each + u * want + (2.0 ** -18 + 2 * 18.4 * 2.0 ** -21) * want


def test_no_keys_at_all_and_repeated_memory():
    q, pk, pv, ck, cv, positions = _inputs(5, 8, 2, 128, 0, 0, torch.bfloat16)
    assert bool((glue.prefix_attention(q, pk, pv, ck, cv, positions) == 0).all())
    q, pk, pv, ck, cv, positions = _inputs(5, 8, 2, 128, 100, 30, torch.bfloat16)
    once = ck[:1].expand(5, -1, -1, -1)  # every row's cache the same memory: a stride of 0
    with pytest.raises(ValueError, match="strides"):
        glue.prefix_attention(q, pk, pv, once, cv, positions)
    # of a dimension of one the stride is not read, whatever it is
    got = glue.prefix_attention(q[:1], pk, pv, ck[:1].as_strided(ck[:1].shape, (3, *ck.stride()[1:])), cv[:1], positions[:1])
    assert torch.equal(got, glue.prefix_attention(q[:1], pk, pv, ck[:1], cv[:1], positions[:1]))


def test_more_pieces_than_16_bits_count():
    """65536 rows of 300 KV heads, one key each: 66419 pieces a group of each of 148 blocks.  With one
    key its weight is 1 and the result its value."""
    batch, heads = 65536, 300
    q = torch.zeros(batch, heads, 64, device="cuda", dtype=torch.bfloat16)
    ck = torch.zeros(batch, heads, 1, 64, device="cuda", dtype=torch.bfloat16)
    cv = torch.empty_like(ck).normal_()
    none = torch.zeros(heads, 0, 64, device="cuda", dtype=torch.bfloat16)
    got = glue.prefix_attention(q, none, none, ck, cv, torch.zeros(batch, dtype=torch.long, device="cuda"))
    assert torch.equal(got, cv.view(batch, heads * 64))
    del q, ck, cv, got
    torch.cuda.empty_cache()
