"""Frequencies of rotary positions, with the scalings that models trained on short contexts use on
long ones.  Plain Python in f64: the kernels (`glue.rotary`, `glue.rotary_cache`, `glue.rotary_table`)
take the numbers, whatever rule made them."""

from __future__ import annotations

import math
from dataclasses import dataclass


@dataclass(frozen=True)
class RopeScaling:
    """How the frequencies of a model trained on `original_positions` positions are changed for
    `factor` times as many.

    * "linear": every frequency divided by `factor`.
    * "ntk": theta raised to theta * factor^(d / (d - 2)): the last pair turns `factor` times slower,
      the first as before.
    * "llama3": pairs that turn more than `high` times within the original context keep their
      frequency, those that turn less than `low` times have it divided by `factor`, and between them
      the two are mixed, linearly in the number of turns.
    * "yarn": the same mixture, linear in the pair's index, between the indices of `beta_fast` and of
      `beta_slow` turns; cosines and sines are multiplied by `attention_factor`
      (0.1 ln(factor) + 1 unless given), which scales the scores by its square.
    """

    kind: str
    factor: float
    original_positions: int = 8192
    low: float = 1.0
    high: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self) -> None:
        if self.kind not in ("linear", "ntk", "llama3", "yarn"):
            raise ValueError(f"rope scaling is 'linear', 'ntk', 'llama3' or 'yarn', not {self.kind!r}")
        if not self.factor >= 1.0:
            raise ValueError(f"rope scaling: a factor of {self.factor} does not lengthen the context")
        if self.original_positions < 1:
            raise ValueError(f"rope scaling: {self.original_positions} original positions")
        if self.kind == "llama3" and not 0.0 < self.low < self.high:
            raise ValueError(f"rope scaling: low {self.low} and high {self.high} are no interval")
        if self.kind == "yarn" and not 0.0 < self.beta_slow < self.beta_fast:
            raise ValueError(f"rope scaling: beta_slow {self.beta_slow} and beta_fast {self.beta_fast} are no interval")


def frequencies(rotary_dim: int, theta: float, scaling: RopeScaling | None = None) -> tuple[list[float], float]:
    """Radians a position turns each of the `rotary_dim / 2` pairs by, and the factor on cosine and sine."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary positions turn pairs: {rotary_dim} numbers of a head are none")
    if not theta > 1.0:
        raise ValueError(f"rotary positions: theta is more than 1, not {theta}")
    plain = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return plain, 1.0
    factor = float(scaling.factor)
    if scaling.kind == "linear":
        return [f / factor for f in plain], 1.0
    if scaling.kind == "ntk":
        if rotary_dim == 2:
            return plain, 1.0  # one pair, of frequency 1 whatever theta is
        base = theta * factor ** (rotary_dim / (rotary_dim - 2.0))
        return [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)], 1.0
    if scaling.kind == "llama3":
        out = []
        for f in plain:
            turns = scaling.original_positions * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - scaling.low) / (scaling.high - scaling.low)))
            out.append(f * (keep + (1.0 - keep) / factor))
        return out, 1.0

    def index(turns: float) -> float:  # of the pair that turns so often within the original context
        return rotary_dim * math.log(scaling.original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    first = max(0, math.floor(index(scaling.beta_fast)))
    last = min(rotary_dim - 1, math.ceil(index(scaling.beta_slow)))
    out = []
    for i, f in enumerate(plain):
        ramp = min(1.0, max(0.0, (i - first) / max(0.001, last - first)))
        out.append(f * ((1.0 - ramp) + ramp / factor))
    attention = scaling.attention_factor
    return out, float(0.1 * math.log(factor) + 1.0 if attention is None else attention)
