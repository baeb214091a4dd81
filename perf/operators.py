"""The operators of a decode step that go with sampling many answers to one prompt, as cases that can
be timed and compared: rotary positions (of a prompt, and of one token a row with its cache write),
attention of a batch over one shared prefix and each row's own cache, and the log probabilities of
given tokens with entropy and top alternatives.

`listed()` are fixed cases, `draw(rng)` gives others of the same ranges.  `prepare` makes what a
program holds before the call, `run` is one pass: in elementary torch operations, or with `own` set
through the package's entry points.  `work` is what a pass cannot do without, `exact` the results in
64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_MAX_PREFIX_FLOPS = 4.0 * 256 * 32 * 128 * (16384 + 64.5)
_MAX_LOGITS = 2048 * 128256


def listed() -> list[dict]:
    return [
        # The step of one sequence: the fused projection of an 8B-shaped layer, halves rotated, with
        # the long-context scaling of that model family.  The smallest call: latency.
        {"name": "rotary_cache_1", "op": "rotary_cache", "rows": 1, "nq": 32, "nkv": 8, "hd": 128, "rotary": 128,
         "layout": "half", "scaling": "llama3", "dtype": "bf16", "slots": 2048, "offset": 0},
        # A serving batch of sequences behind a shared prompt; neighbouring pairs of half the head rotated.
        {"name": "rotary_cache_61_pairs_f16", "op": "rotary_cache", "rows": 61, "nq": 32, "nkv": 8, "hd": 128, "rotary": 64,
         "layout": "interleaved", "scaling": "none", "dtype": "f16", "slots": 512, "offset": 100003},
        # A prompt of 8192 tokens through an 8B-shaped layer.
        {"name": "rotary_8192", "op": "rotary", "tokens": 8192, "nq": 32, "nkv": 8, "hd": 128, "rotary": 128,
         "layout": "half", "scaling": "llama3", "dtype": "bf16", "start": 0},
        # A chunk from the middle of a very long context, an odd number of tokens, neighbouring pairs, f16.
        {"name": "rotary_1021_pairs_far_f16", "op": "rotary", "tokens": 1021, "nq": 28, "nkv": 4, "hd": 128, "rotary": 128,
         "layout": "interleaved", "scaling": "yarn", "dtype": "f16", "start": 1000003},
        # Two answers to a short question by a small model: latency.
        {"name": "prefix_2x100", "op": "prefix", "rows": 2, "nq": 4, "nkv": 2, "hd": 64, "prefix": 100, "own_keys": 5, "dtype": "bf16"},
        # 64 samples of one 8192-token prompt, up to 512 tokens into their answers, 8B-shaped heads.
        {"name": "prefix_64x8192", "op": "prefix", "rows": 64, "nq": 32, "nkv": 8, "hd": 128, "prefix": 8192, "own_keys": 512, "dtype": "bf16"},
        # An odd batch over an odd prefix, seven heads to a KV head, heads of 64, f16.
        {"name": "prefix_33x5001_f16", "op": "prefix", "rows": 33, "nq": 14, "nkv": 2, "hd": 64, "prefix": 5001, "own_keys": 300, "dtype": "f16"},
        # 256 samples of a 16384-token document, early in their answers: the products count here.
        {"name": "prefix_256x16384", "op": "prefix", "rows": 256, "nq": 32, "nkv": 8, "hd": 128, "prefix": 16384, "own_keys": 128, "dtype": "bf16"},
        # The token just sampled, with the 20 alternatives an API offers: latency.
        {"name": "logprobs_1_top20", "op": "logprobs", "rows": 1, "vocab": 128256, "top": 20, "masked": 0.0, "dtype": "bf16"},
        # A decode batch under a grammar that forbids nine tokens in ten, logits kept in f32.
        {"name": "logprobs_64_masked_f32", "op": "logprobs", "rows": 64, "vocab": 128256, "top": 5, "masked": 0.9, "dtype": "f32"},
        # A vocabulary of an odd size in f16, no alternatives asked for.
        {"name": "logprobs_333_odd_f16", "op": "logprobs", "rows": 333, "vocab": 32003, "top": 0, "masked": 0.0, "dtype": "f16"},
        # Scoring a chunk of 2048 prompt tokens.
        {"name": "logprobs_2048_top5", "op": "logprobs", "rows": 2048, "vocab": 128256, "top": 5, "masked": 0.0, "dtype": "bf16"},
    ]


def _log(rng: random.Random, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["rotary", "rotary_cache", "prefix", "prefix", "prefix", "logprobs", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "logprobs":
        rows = _log(rng, 1, 2048)
        vocab = min(_log(rng, 1000, 200000), _MAX_LOGITS // rows)
        dtype = rng.choice(["bf16", "f16", "f32"])
        if dtype == "f32":
            rows = (rows + 1) // 2
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, rng.randint(2, 20), 20]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99]), "dtype": dtype}
    nkv = rng.choice([1, 2, 4, 8])
    rep = rng.choice([1, 2, 4, 4, 4, 7, 8]) if nkv < 8 else rng.choice([1, 2, 4])
    if op == "prefix":
        hd = rng.choice([64, 128, 128])
        rows, own_keys = _log(rng, 1, 256), _log(rng, 1, 1000)
        prefix = _log(rng, 16, 32768)
        prefix = max(1, min(prefix, int(_MAX_PREFIX_FLOPS / (4.0 * rows * nkv * rep * hd)) - own_keys))
        return {"op": op, "rows": rows, "nq": nkv * rep, "nkv": nkv, "hd": hd, "prefix": prefix, "own_keys": own_keys, "dtype": dtype}
    hd = rng.choice([64, 128])
    shape = {"op": op, "nq": nkv * rep, "nkv": nkv, "hd": hd, "rotary": rng.choice([hd, hd, hd // 2, hd - 16]),
             "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "dtype": dtype}
    if op == "rotary":
        return {**shape, "tokens": _log(rng, 1, 8192), "start": rng.choice([0, _log(rng, 1, 1000000)])}
    return {**shape, "rows": _log(rng, 1, 256), "slots": _log(rng, 16, 600), "offset": rng.choice([0, _log(rng, 1, 100000)])}


# ---- what a program holds before the call ---------------------------------------------------


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape: tuple[int, ...], std: float, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)


def _frequencies(rotary: int, scaling: str) -> tuple[list[float], float]:
    """Radians a position turns each pair by, and the factor on cosine and sine, of a model trained on
    8192 positions and used on more."""
    theta, original = 500000.0, 8192.0
    plain = [theta ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if scaling == "linear":
        return [f / 4.0 for f in plain], 1.0
    if scaling == "llama3":  # long wavelengths divided by 8, short ones kept, a ramp between
        out = []
        for f in plain:
            turns = original * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            out.append(f * (keep + (1.0 - keep) / 8.0))
        return out, 1.0
    if scaling == "yarn":  # by the pair's index between 32 turns and 1, and the factor that goes with it
        index = [rotary * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(0, math.floor(index[0])), min(rotary - 1, math.ceil(index[1]))
        out = []
        for i, f in enumerate(plain):
            ramp = min(1.0, max(0.0, (i - low) / max(0.001, high - low)))
            out.append(f * ((1.0 - ramp) + ramp / 16.0))
        return out, 0.1 * math.log(16.0) + 1.0
    return plain, 1.0


def _newest(case: dict) -> list[int]:
    """Slot of each row's newest key in its own cache: the last one for the first row, others spread
    over the whole range; now and then a row that has none of its own yet."""
    keys = case["own_keys"]
    return [keys - 1] + [(i * 7919) % (keys + 1) - 1 for i in range(1, case["rows"])]


def prepare(case: dict, seed: int) -> dict:
    op, gen, dtype = case["op"], _generator(seed), _DTYPES[case["dtype"]]
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal((rows, vocab), 2.5, dtype, gen)
        if case["masked"]:  # a tenth of the rows has a token forbidden that was given all the same
            logits.masked_fill_(torch.rand(rows, vocab, device="cuda", generator=gen) < case["masked"], -math.inf)
        tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        if case["masked"]:
            likely = logits.argmax(dim=-1)
            tokens = torch.where(torch.arange(rows, device="cuda") % 10 == 9, tokens, likely)
        return {"op": op, "logits": logits, "tokens": tokens, "top": case["top"]}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if op == "prefix":
        rows, prefix, keys = case["rows"], case["prefix"], case["own_keys"]
        room = 64 * ((prefix + 63) // 64)  # the prompt's cache was laid out for a little more than the prompt
        prompt = _normal((2, nkv, room, hd), 1.0, dtype, gen)
        cache = _normal((2, rows, nkv, keys, hd), 1.0, dtype, gen)
        return {"op": op, "q": _normal((rows, nq, hd), 1.5, dtype, gen), "prefix_k": prompt[0][:, :prefix],
                "prefix_v": prompt[1][:, :prefix], "cache_k": cache[0], "cache_v": cache[1],
                "positions": torch.tensor(_newest(case), device="cuda", dtype=torch.long)}
    freq, factor = _frequencies(case["rotary"], case["scaling"])
    state = {"op": op, "nq": nq, "nkv": nkv, "hd": hd, "layout": case["layout"], "factor": factor,
             "frequencies": torch.tensor(freq, device="cuda", dtype=torch.float64)}
    if op == "rotary":
        tokens = case["tokens"]
        qkv = _normal((tokens, nq + 2 * nkv, hd), 1.0, dtype, gen)  # the fused projection: q and k are views of it
        return {**state, "q": qkv[:, :nq], "k": qkv[:, nq:nq + nkv],
                "positions": torch.arange(case["start"], case["start"] + tokens, device="cuda", dtype=torch.long)}
    rows, slots = case["rows"], case["slots"]
    return {**state, "qkv": _normal((rows, (nq + 2 * nkv) * hd), 1.0, dtype, gen), "offset": case["offset"],
            "cache_k": torch.zeros(rows, nkv, slots, hd, device="cuda", dtype=dtype),
            "cache_v": torch.zeros(rows, nkv, slots, hd, device="cuda", dtype=dtype),
            "positions": torch.tensor([slots - 1 - (i * 37) % slots for i in range(rows)], device="cuda", dtype=torch.long)}


# ---- one pass ---------------------------------------------------------------------------------


def _rotated(x: torch.Tensor, angle: torch.Tensor, layout: str, factor: float) -> torch.Tensor:
    """x [tokens, heads, D] with its first 2 * pairs numbers of a head turned by angle [tokens, pairs] (f64)."""
    pairs = angle.shape[-1]
    cos, sin = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    head, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    if layout == "half":
        a, b = head[..., :pairs], head[..., pairs:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), rest], dim=-1)


def _plain_rotary(s: dict):
    angle = s["positions"].double()[:, None] * s["frequencies"][None]
    return _rotated(s["q"], angle, s["layout"], s["factor"]), _rotated(s["k"], angle, s["layout"], s["factor"])


def _plain_rotary_cache(s: dict):
    nq, nkv, slots = s["nq"], s["nkv"], s["positions"]
    qkv = s["qkv"].view(-1, nq + 2 * nkv, s["hd"])
    angle = (slots + s["offset"]).double()[:, None] * s["frequencies"][None]
    rows = torch.arange(qkv.shape[0], device=qkv.device)
    s["cache_k"][rows, :, slots] = _rotated(qkv[:, nq:nq + nkv], angle, s["layout"], s["factor"])
    s["cache_v"][rows, :, slots] = qkv[:, nq + nkv:]
    return _rotated(qkv[:, :nq], angle, s["layout"], s["factor"]), s["cache_k"], s["cache_v"]


def _plain_prefix(s: dict):
    q, prefix_k, cache_k = s["q"], s["prefix_k"].float(), s["cache_k"].float()
    rows, nq, hd = q.shape
    nkv, prefix = prefix_k.shape[:2]
    grouped = q.float().view(rows, nkv, nq // nkv, hd) / math.sqrt(hd)
    shared = torch.einsum("bgrd,gpd->bgrp", grouped, prefix_k)
    alone = torch.einsum("bgrd,bgsd->bgrs", grouped, cache_k)
    behind = torch.arange(cache_k.shape[2], device=q.device)[None] > s["positions"][:, None]
    alone.masked_fill_(behind[:, None, None], -math.inf)
    scores = torch.cat([shared, alone], dim=-1)
    weights = (scores - scores.amax(dim=-1, keepdim=True)).exp()
    out = torch.einsum("bgrp,gpd->bgrd", weights[..., :prefix], s["prefix_v"].float())
    out += torch.einsum("bgrs,bgsd->bgrd", weights[..., prefix:], s["cache_v"].float())
    return (out / weights.sum(dim=-1, keepdim=True)).to(q.dtype).reshape(rows, nq * hd)


def _plain_logprobs(s: dict):
    x, tokens, top = s["logits"].float(), s["tokens"], s["top"]
    shifted = x - x.amax(dim=-1, keepdim=True)
    weights = shifted.exp()
    total = weights.sum(dim=-1, dtype=torch.float64)
    mean = (weights * shifted.clamp_min(-1e4)).sum(dim=-1, dtype=torch.float64) / total
    norm = total.log()
    given = (shifted.gather(1, tokens[:, None])[:, 0].double() - norm).float()
    entropy = (norm - mean).float()
    if not top:
        return given, entropy
    # one whole number a logit: its order among floats, then the lower index first
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    behind = torch.arange(x.shape[1], device=x.device)
    key = order * (1 << 32) + ((1 << 32) - 1 - behind)
    index = ((1 << 32) - 1) - (key.topk(top, dim=-1).values & 0xFFFFFFFF)
    return given, entropy, (shifted.gather(1, index).double() - norm[:, None]).float(), index


def run(state: dict):
    op = state["op"]
    if not own:
        return {"rotary": _plain_rotary, "rotary_cache": _plain_rotary_cache, "prefix": _plain_prefix,
                "logprobs": _plain_logprobs}[op](state)
    from linnet_b200 import glue

    s = state
    if op == "rotary":
        return glue.rotary(s["q"], s["k"], s["positions"], s["frequencies"], layout=s["layout"], factor=s["factor"])
    if op == "rotary_cache":
        q = glue.rotary_cache(s["qkv"], s["positions"], s["frequencies"], s["cache_k"], s["cache_v"], s["nq"], s["nkv"],
                              layout=s["layout"], factor=s["factor"], offset=s["offset"])
        return q, s["cache_k"], s["cache_v"]
    if op == "prefix":
        return glue.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["cache_k"], s["cache_v"], s["positions"])
    got = glue.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    return tuple(got) if s["top"] else tuple(got)[:2]


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case: dict) -> dict:
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        # subtract, exponential, two sums and a product; a comparison for the alternatives
        return {"bytes": rows * (vocab * size + 8.0 + 8.0 + 12.0 * top), "flops": rows * vocab * (6.0 + (top > 0))}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if op == "prefix":
        rows, prefix = case["rows"], case["prefix"]
        keys = sum(p + 1 for p in _newest(case))
        return {"bytes": 2.0 * size * nkv * hd * (prefix + keys) + 2.0 * size * rows * nq * hd + 8.0 * rows,
                "flops": 4.0 * nq * hd * (rows * prefix + keys)}
    if op == "rotary":
        return {"bytes": case["tokens"] * (2.0 * size * (nq + nkv) * hd + 8.0), "flops": 3.0 * case["tokens"] * (nq + nkv) * case["rotary"]}
    return {"bytes": case["rows"] * (2.0 * size * (nq + 2 * nkv) * hd + 8.0), "flops": 3.0 * case["rows"] * (nq + nkv) * case["rotary"]}


# ---- the same results in 64 bits ------------------------------------------------------------------


def _exact_turn(x: torch.Tensor, positions: torch.Tensor, s: dict) -> torch.Tensor:
    """Pairs as complex numbers times factor * e^(i * position * frequency)."""
    turn = torch.polar(torch.full_like(s["frequencies"], s["factor"]).expand(len(positions), -1),
                       positions.double().outer(s["frequencies"]))[:, None]
    pairs, out = turn.shape[-1], x.double()
    if s["layout"] == "half":
        at = torch.arange(pairs, device=x.device)
        first, second = at, at + pairs
    else:
        at = 2 * torch.arange(pairs, device=x.device)
        first, second = at, at + 1
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        return _exact_turn(s["q"], s["positions"], s), _exact_turn(s["k"], s["positions"], s)
    if op == "rotary_cache":
        nq, nkv = s["nq"], s["nkv"]
        heads = s["qkv"].unflatten(-1, (nq + 2 * nkv, s["hd"]))
        turned = _exact_turn(heads[:, :nq + nkv], s["positions"] + s["offset"], s)
        keys, values = s["cache_k"].double(), s["cache_v"].double()
        for row, slot in enumerate(s["positions"].tolist()):
            keys[row, :, slot] = turned[row, nq:]
            values[row, :, slot] = heads[row, nq + nkv:].double()
        return turned[:, :nq].contiguous(), keys, values
    if op == "prefix":
        nkv, rep = case["nkv"], case["nq"] // case["nkv"]
        out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
        newest = s["positions"].tolist()
        for group in range(nkv):
            shared_k, shared_v = s["prefix_k"][group].double(), s["prefix_v"][group].double()
            for row, last in enumerate(newest):
                heads = slice(group * rep, (group + 1) * rep)
                keys = torch.cat([shared_k, s["cache_k"][row, group, :last + 1].double()])
                values = torch.cat([shared_v, s["cache_v"][row, group, :last + 1].double()])
                scores = s["q"][row, heads].double() @ keys.T * case["hd"] ** -0.5
                out[row, heads] = torch.softmax(scores, dim=-1) @ values
        return out.flatten(1)
    given, entropy, best, index = [], [], [], []
    for begin in range(0, case["rows"], 256):
        logits = s["logits"][begin:begin + 256].double()
        logprob = logits - torch.logsumexp(logits, dim=-1, keepdim=True)
        given.append(logprob.gather(1, s["tokens"][begin:begin + 256, None])[:, 0])
        entropy.append(-torch.special.xlogy(logprob.exp(), logprob.exp()).sum(dim=-1))
        if case["top"]:
            order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            best.append(logprob.gather(1, order))
            index.append(order)
    whole = (given, entropy, best, index) if case["top"] else (given, entropy)
    return tuple(torch.cat(part) for part in whole)
