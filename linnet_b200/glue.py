"""PyTorch-facing wrappers of the decode-step glue kernels (`csrc/decoder_glue.cu`):
residual add + RMSNorm, rotary embedding + KV-cache write, single-query attention over
the cache, and SwiGLU's `silu(gate) * up`.  bf16 CUDA tensors only; launches go to the
current stream and record into CUDA graphs.

For many answers to one prompt, bf16 or f16: rotary positions of any frequencies, layout and part
of a head (`csrc/rotary.cu`: `rotary`, `rotary_cache`, `rotary_table`; `rope_frequencies` makes the
frequencies), attention over one shared prefix and each row's own cache
(`csrc/prefix_attention.cu`: `prefix_attention`), and log probabilities of given tokens with entropy
and alternatives (`csrc/token_logprobs.cu`: `token_logprobs`).  These have no derivative and refuse
tensors that ask for one, in reverse or in forward mode."""

from __future__ import annotations

import functools
import operator
import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib, rope
from .kernels import _CODES, _current_device, _raw_stream


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _bf16(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise RuntimeError("glue kernels take contiguous bf16 CUDA tensors")


def _positions(positions: torch.Tensor, batch: int, device: torch.device) -> None:
    """Positions are read on the device as int64: anything else would be misread."""
    if (not positions.is_cuda or positions.device != device or positions.dtype != torch.int64
            or not positions.is_contiguous() or positions.numel() != batch):
        raise ValueError(f"positions must be a contiguous int64 tensor of {batch} entries on {device}, not "
                         f"{positions.dtype}{list(positions.shape)} on {positions.device}")


def decoder_status() -> None:
    """Raises if a decode-step kernel met a position outside its cache since the last call
    (synchronises the device; `b200q_decoder_status`)."""
    _lib.check(_lib.load().b200q_decoder_status())


def add_rmsnorm(x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """`x += delta` in place (when given), returns `rms_norm(x) * weight`."""
    _bf16(x, weight, *([] if delta is None else [delta]))
    rows, hidden = x.shape
    y = torch.empty_like(x)
    _lib.check(_lib.load().b200q_add_rmsnorm(x.data_ptr(), None if delta is None else delta.data_ptr(),
                                             weight.data_ptr(), y.data_ptr(), rows, hidden, eps, _stream(x)))
    return y


def rope_cache(qkv: torch.Tensor, positions: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
               nq: int, nkv: int, theta: float) -> torch.Tensor:
    """Rotates q and k of `qkv` [B, (nq + 2 nkv) * D], writes k and v into the caches
    [B, nkv, S, D] at `positions` and returns q [B, nq, D]."""
    _bf16(qkv, cache_k, cache_v)
    batch = qkv.shape[0]
    _positions(positions, batch, qkv.device)
    _, _, max_seq, hd = cache_k.shape
    q = torch.empty(batch, nq, hd, device=qkv.device, dtype=qkv.dtype)
    _lib.check(_lib.load().b200q_rope_cache(qkv.data_ptr(), positions.data_ptr(), q.data_ptr(),
                                            cache_k.data_ptr(), cache_v.data_ptr(), batch, nq, nkv, hd,
                                            max_seq, theta, _stream(qkv)))
    return q


def attention_splits(batch: int, nkv: int, max_seq: int, sms: int = 148) -> int:
    """Key splits (a power of two, at least 64 positions each) for about two blocks per
    multiprocessor: measured on a B200 at 2048 positions, batch 1 is fastest with 8 splits,
    batch 8 with 4, batch 64 with 1."""
    want = max(1, (2 * sms) // max(1, batch * nkv))
    splits = 1
    while splits * 2 <= want and max_seq // (splits * 2) >= 64:
        splits *= 2
    return splits


def decode_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                     positions: torch.Tensor, splits: int | None = None) -> torch.Tensor:
    """Attention of one query per row, q [B, nq, D], over cache positions 0..positions[b];
    returns [B, nq * D].  Up to 8 key splits run as one launch (the splits of a row and KV
    head are a thread-block cluster); more need a scratch tensor and a second, merging launch."""
    _bf16(q, cache_k, cache_v)
    batch, nq, hd = q.shape
    _positions(positions, batch, q.device)
    _, nkv, max_seq, _ = cache_k.shape
    if splits is None:
        splits = min(8, attention_splits(batch, nkv, max_seq))
    lib = _lib.load()
    out = torch.empty(batch, nq * hd, device=q.device, dtype=q.dtype)
    if splits <= 8:
        _lib.check(lib.b200q_decode_attention_cluster(q.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(),
                                                      positions.data_ptr(), out.data_ptr(), batch, nq, nkv, hd,
                                                      max_seq, splits, _stream(q)))
        return out
    scratch = torch.empty(lib.b200q_decode_attention_scratch_bytes(batch, nq, hd, splits), dtype=torch.uint8,
                          device=q.device)
    _lib.check(lib.b200q_decode_attention(q.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(),
                                          positions.data_ptr(), out.data_ptr(), scratch.data_ptr(), batch, nq,
                                          nkv, hd, max_seq, splits, _stream(q)))
    return out


def rope_table(max_seq: int, head_dim: int, theta: float, device: torch.device) -> torch.Tensor:
    """(cos, sin) of every position and frequency, f32 [max_seq, head_dim / 2, 2], for `rope_attention`."""
    table = torch.empty(max_seq, head_dim // 2, 2, dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _lib.check(_lib.load().b200q_rope_table(table.data_ptr(), max_seq, head_dim, float(theta),
                                                torch.cuda.current_stream(device).cuda_stream))
    return table


def rope_attention(qkv: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, cache_k: torch.Tensor,
                   cache_v: torch.Tensor, nq: int, nkv: int, splits: int | None = None) -> torch.Tensor:
    """`rope_cache` + `decode_attention` in one launch: rotates q and k of the fused projection
    qkv [B, (nq + 2 nkv) * D] at positions[b], appends k and v to the caches and attends over
    positions 0..positions[b]; returns [B, nq * D]."""
    _bf16(qkv, cache_k, cache_v)
    batch, _, max_seq, hd = cache_k.shape
    _positions(positions, batch, qkv.device)
    if splits is None:
        splits = min(8, attention_splits(batch, nkv, max_seq))
    if table.shape != (max_seq, hd // 2, 2) or table.dtype != torch.float32:
        raise ValueError("rope_attention: the table does not match the cache")
    out = torch.empty(batch, nq * hd, device=qkv.device, dtype=qkv.dtype)
    _lib.check(_lib.load().b200q_rope_attention(qkv.data_ptr(), positions.data_ptr(), table.data_ptr(),
                                                cache_k.data_ptr(), cache_v.data_ptr(), out.data_ptr(), batch, nq,
                                                nkv, hd, max_seq, splits, _stream(qkv)))
    return out


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """`silu(gate_up[:, :I]) * gate_up[:, I:]` for gate_up [B, 2 I]."""
    _bf16(gate_up)
    rows, width = gate_up.shape
    out = torch.empty(rows, width // 2, device=gate_up.device, dtype=gate_up.dtype)
    _lib.check(_lib.load().b200q_silu_mul(gate_up.data_ptr(), out.data_ptr(), rows, width // 2, _stream(gate_up)))
    return out


# ---- many answers to one prompt --------------------------------------------------------------

_LAYOUTS = {"half": 0, "interleaved": 1}
_strides_of = struct.Struct("12q").pack


def _same(who: str, kinds: tuple[torch.dtype, ...], *tensors: torch.Tensor) -> int:
    """One CUDA device (returned), one of `kinds`, last dimension contiguous, no derivative asked for."""
    first = tensors[0]
    index, kind = first.get_device(), first.dtype
    for t in tensors:
        if t.get_device() != index or index < 0 or t.dtype is not kind or kind not in kinds:
            names = ", ".join(str(k).removeprefix("torch.") for k in kinds)
            raise RuntimeError(f"{who} takes CUDA tensors of one device and one of the types {names}; got "
                               f"{[f'{t.dtype} on {t.device}' for t in tensors]}")
        if not t.is_contiguous() and t.stride(-1) != 1 and t.numel() > 0 and t.shape[-1] > 1:
            raise RuntimeError(f"{who}: the last dimension has to be contiguous")
        if t.requires_grad or forward_ad._current_level >= 0:
            _no_derivative(who, t)
    return index


def _no_derivative(who: str, t: torch.Tensor) -> None:
    """Of a tensor that may ask for one.  (A forward-mode tangent counts under torch.no_grad() too, which leaves that
    mode on.)"""
    if (t.requires_grad and torch.is_grad_enabled()) or forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{who} has no derivative: detach its inputs or call it under torch.no_grad()")


def _launch(index: int, entry, *args) -> None:
    """Calls an entry of the library on the device's current stream.  A call of the smallest sizes is
    bound by its host path: no context manager unless another device is current."""
    if index == _current_device():
        status = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _raw_stream(index))
    if status:
        _lib.check(status)


def _words(who: str, name: str, words: torch.Tensor, count: int, index: int) -> None:
    """Read on the device as int64: anything else would be misread."""
    if (words.get_device() != index or words.dtype is not torch.int64 or words.numel() != count
            or not words.is_contiguous()):
        raise ValueError(f"{who}: {name} must be a contiguous int64 tensor of {count} entries on cuda:{index}, not "
                         f"{words.dtype}{list(words.shape)} on {words.device}")


_HALF = (torch.bfloat16, torch.float16)
_LOGITS = (torch.bfloat16, torch.float16, torch.float32)


def _contiguous(who: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_contiguous():
            raise RuntimeError(f"{who} takes contiguous caches and projections")


def _frequencies(who: str, frequencies: torch.Tensor, head_dim: int, index: int) -> int:
    """Read on the device as f64: anything else would be misread."""
    pairs = frequencies.numel()
    if (frequencies.get_device() != index or frequencies.dtype is not torch.float64 or not frequencies.is_contiguous()
            or frequencies.dim() != 1 or not 1 <= pairs <= head_dim // 2):
        raise ValueError(f"{who}: frequencies must be a contiguous float64 tensor of 1 to {head_dim // 2} entries on "
                         f"cuda:{index}, not {frequencies.dtype}{list(frequencies.shape)} on {frequencies.device}")
    if frequencies.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(who, frequencies)
    return pairs


def _layout(who: str, layout: str) -> int:
    if layout not in _LAYOUTS:
        raise ValueError(f"{who}: layout is 'half' or 'interleaved', not {layout!r}")
    return _LAYOUTS[layout]


def _word(who: str, name: str, value: "int | torch.Tensor", index: int) -> tuple[int | None, int]:
    """A number known on the host, or one int64 word on the device: (address or None, number)."""
    if not isinstance(value, torch.Tensor):
        return None, operator.index(value)
    _words(who, name, value, 1, index)
    return value.data_ptr(), 0


def rope_frequencies(rotary_dim: int, theta: float, *, scaling: "rope.RopeScaling | None" = None,
                     device: "torch.device | str" = "cuda") -> tuple[torch.Tensor, float]:
    """Frequencies f64 [rotary_dim / 2] on `device` and the factor on cosine and sine, for `rotary`,
    `rotary_cache` and `rotary_table` (`rope.RopeScaling` says which scalings there are)."""
    numbers, factor = rope.frequencies(rotary_dim, theta, scaling)
    return torch.tensor(numbers, dtype=torch.float64, device=device), factor


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *,
           layout: str = "half", factor: float = 1.0,
           out: "tuple[torch.Tensor, torch.Tensor | None] | None" = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary positions of a prompt: q [T, nq, D] and k [T, nkv, D] (or None), bf16 or f16, rows and
    heads at any stride (views of a fused projection).  The first `2 * len(frequencies)` numbers of
    every head, as pairs of the two halves ("half") or of neighbours ("interleaved"), are turned by
    positions[t] * frequencies[pair] and multiplied by `factor`; the others are copied.  `out`: where
    the results go, (q, k) themselves to turn in place; other overlaps are not allowed."""
    tensors = (q,) if k is None else (q, k)
    index = _same("rotary", _HALF, *tensors)
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError(f"rotary: q is [tokens, heads, D] and k the same, not {[list(t.shape) for t in tensors]}")
    tokens, nq, hd = q.shape
    _words("rotary", "positions", positions, tokens, index)
    pairs = _frequencies("rotary", frequencies, hd, index)
    code = _layout("rotary", layout)
    if out is None:
        device = q.device
        q_out, k_out = torch.empty(tokens, nq, hd, dtype=q.dtype, device=device), None
        if k is not None:
            k_out = torch.empty(tokens, k.shape[1], hd, dtype=k.dtype, device=device)
    else:
        q_out, k_out = out
        if q_out.shape != q.shape or (k is None) != (k_out is None) or (k is not None and k_out.shape != k.shape):
            raise ValueError("rotary: out has to have the shapes of q and k")
        _same("rotary", _HALF, q, q_out, *(() if k is None else (k_out,)))
    q_from, q_to = q.stride(), q_out.stride()
    keys, k_from, k_to, nkv, at = None, q_from, q_to, 0, None
    if k is not None:
        keys, k_from, k_to, nkv, at = k.data_ptr(), k.stride(), k_out.stride(), k.shape[1], k_out.data_ptr()
    _launch(index, _lib.load().b200q_rotary,
            q.data_ptr(), keys, positions.data_ptr(), frequencies.data_ptr(), q_out.data_ptr(), at, tokens, nq, nkv, hd,
            pairs, q_from[0], q_from[1], k_from[0], k_from[1], q_to[0], q_to[1], k_to[0], k_to[1], factor, code,
            _CODES[q.dtype])
    return q_out, k_out


def rotary_cache(qkv: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, cache_k: torch.Tensor,
                 cache_v: torch.Tensor, nq: int, nkv: int, *, layout: str = "half", factor: float = 1.0,
                 offset: "int | torch.Tensor" = 0) -> torch.Tensor:
    """`rope_cache` with the positions of `rotary`, bf16 or f16: turns q and k of qkv
    [B, (nq + 2 nkv) * D] by (positions[b] + offset) * frequencies, writes k and v into the caches
    [B, nkv, S, D] at slot positions[b] and returns q [B, nq, D].  `offset` (a number, or one int64 on
    the device) is where a row's own cache begins: the length of the prefix it shares.  A position
    outside the cache stores nothing and is reported by `decoder_status`."""
    index = _same("rotary_cache", _HALF, qkv, cache_k, cache_v)
    _contiguous("rotary_cache", qkv, cache_k, cache_v)
    shape = cache_k.shape
    batch, _, max_seq, hd = shape if len(shape) == 4 else (-1, -1, -1, -1)
    if shape != cache_v.shape or shape != (batch, nkv, max_seq, hd) or qkv.shape != (batch, (nq + 2 * nkv) * hd):
        raise ValueError(f"rotary_cache: qkv {list(qkv.shape)} of {nq} and {nkv} heads and caches "
                         f"{list(cache_k.shape)}, {list(cache_v.shape)} do not go together")
    _words("rotary_cache", "positions", positions, batch, index)
    pairs = _frequencies("rotary_cache", frequencies, hd, index)
    code = _layout("rotary_cache", layout)
    at, number = _word("rotary_cache", "offset", offset, index)
    q = torch.empty(batch, nq, hd, device=qkv.device, dtype=qkv.dtype)
    _launch(index, _lib.load().b200q_rotary_cache,
            qkv.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), at, number, q.data_ptr(), cache_k.data_ptr(),
            cache_v.data_ptr(), batch, nq, nkv, hd, pairs, max_seq, factor, code, _CODES[qkv.dtype])
    return q


def rotary_table(max_seq: int, frequencies: torch.Tensor, factor: float = 1.0) -> torch.Tensor:
    """(cos, sin) * factor of positions 0 .. max_seq - 1, f32 [max_seq, len(frequencies), 2]: what
    `rope_attention` takes, for frequencies of any scaling (of whole heads, halves turned)."""
    if not frequencies.is_cuda or max_seq < 1:
        raise ValueError(f"rotary_table: {max_seq} positions, frequencies on {frequencies.device}")
    index = frequencies.get_device()
    pairs = _frequencies("rotary_table", frequencies, 1024, index)
    table = torch.empty(max_seq, pairs, 2, dtype=torch.float32, device=frequencies.device)
    _launch(index, _lib.load().b200q_rotary_table, table.data_ptr(), frequencies.data_ptr(), max_seq, pairs, factor)
    return table


@functools.lru_cache(maxsize=256)
def _prefix_scratch(index: int, batch: int, nq: int, nkv: int, head_dim: int, prefix: int, max_seq: int) -> int:
    """Bytes of scratch memory; of the sizes alone (and the device's multiprocessors)."""
    with torch.cuda.device(index):
        size = _lib.load().b200q_prefix_attention_scratch_bytes(batch, nq, nkv, head_dim, prefix, max_seq)
    if size < 0:
        raise ValueError(_lib.last_error())
    return size


def prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, cache_k: torch.Tensor,
                     cache_v: torch.Tensor, positions: torch.Tensor, *, prefix_length: "torch.Tensor | None" = None,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of one query per row, q [B, nq, D], over a prefix that all rows share, keys and values
    [nkv, P, D] (read once for the batch), and then over positions 0..positions[b] of each row's own
    cache [B, nkv, S, D]; returns [B, nq * D].  bf16 or f16, D 64 or 128, nq / nkv up to 128; `scale`, a
    positive number, is D**-0.5 unless given.  A position of -1 is a row without keys of its own; one outside the cache
    counts as that and is reported by `decoder_status`.  `prefix_length`: one int64 on the device, how
    many of the P positions there are (a captured step can be replayed on another prompt).  The last
    dimension is contiguous, other strides are positive multiples of 8 numbers (parts of longer caches)."""
    index = _same("prefix_attention", _HALF, q, prefix_k, prefix_v, cache_k, cache_v)
    shape, shared, own = q.shape, prefix_k.shape, cache_k.shape
    batch, nq, hd = shape if len(shape) == 3 else (-1, -1, -1)
    nkv, prefix = shared[:2] if len(shared) == 3 else (-1, -1)
    if (batch < 0 or shared != (nkv, prefix, hd) or shared != prefix_v.shape or len(own) != 4 or own != cache_v.shape
            or own[0] != batch or own[1] != nkv or own[3] != hd):
        raise ValueError(f"prefix_attention: q {list(shape)}, a prefix {list(shared)}, {list(prefix_v.shape)} and "
                         f"caches {list(own)}, {list(cache_v.shape)} do not go together")
    _words("prefix_attention", "positions", positions, batch, index)
    at = None
    if prefix_length is not None:
        if not isinstance(prefix_length, torch.Tensor):
            raise ValueError("prefix_attention: prefix_length is one int64 on the device (or cut the prefix to its length)")
        at, _ = _word("prefix_attention", "prefix_length", prefix_length, index)
    pk, pv, ck, cv = prefix_k.stride(), prefix_v.stride(), cache_k.stride(), cache_v.stride()
    steps = q.stride()
    strides = _strides_of(steps[0], steps[1], pk[1], pk[0], pv[1], pv[0], ck[2], ck[1], ck[0], cv[2], cv[1], cv[0])
    device, kind = q.device, q.dtype
    scratch = torch.empty(_prefix_scratch(index, batch, nq, nkv, hd, prefix, own[2]), dtype=torch.uint8, device=device)
    out = torch.empty(batch, nq * hd, dtype=kind, device=device)
    _launch(index, _lib.load().b200q_prefix_attention,
            q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(),
            positions.data_ptr(), at, out.data_ptr(), scratch.data_ptr(), batch, nq, nkv, hd, prefix, own[2],
            strides, hd ** -0.5 if scale is None else scale, _CODES[kind])
    return out


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # f32 [rows]: of the tokens given
    entropy: torch.Tensor       # f32 [rows], in nats
    top_logprobs: torch.Tensor  # f32 [rows, top], the most probable first
    top_tokens: torch.Tensor    # int64 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Log probabilities of tokens [rows] under softmax(logits [rows, vocab]), the entropy of every row
    and its `top` (up to 32) most probable tokens with theirs, the lower index first among equals.
    Logits are f32, bf16 or f16, rows at any stride; -inf is a forbidden token.  A negative token
    stands for none (log probability 0: padded rows drop out of sums); one past the vocabulary gives
    NaN and is reported by `decoder_status`."""
    index = _same("token_logprobs", _LOGITS, logits)
    shape = logits.shape
    if len(shape) != 2 or not 0 < shape[1]:
        raise ValueError(f"token_logprobs: logits are [rows, vocab], not {list(shape)}")
    rows, vocab = shape
    if tokens.dim() != 1:
        raise ValueError(f"token_logprobs: tokens must be an int64 tensor [rows], not {tokens.dtype}{list(tokens.shape)}")
    _words("token_logprobs", "tokens", tokens, rows, index)
    if not 0 <= top <= min(32, vocab):
        raise ValueError(f"token_logprobs: 0 to {min(32, vocab)} alternatives of a row, not {top}")
    device = logits.device
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    entropy = torch.empty(rows, dtype=torch.float32, device=device)
    best = torch.empty(rows, top, dtype=torch.float32, device=device)
    best_tokens = torch.empty(rows, top, dtype=torch.int64, device=device)
    _launch(index, _lib.load().b200q_token_logprobs,
            logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), best.data_ptr(),
            best_tokens.data_ptr(), rows, vocab, logits.stride(0), top, _CODES[logits.dtype])
    return TokenLogprobs(logprob, entropy, best, best_tokens)
