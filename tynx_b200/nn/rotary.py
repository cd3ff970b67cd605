"""Rotary position frequencies."""

from __future__ import annotations

import math
from typing import Optional

import numpy as np

from .. import _native as N


class Rotary:
    """The rotation of a head's first ``dim`` elements by a token's position:
    pair ``i`` of the ``dim / 2`` turns by ``position * frequencies[i]`` radians,
    ``frequencies[i] = base ** (-2 i / dim)`` before scaling.  Pairs are elements
    ``(i, i + dim / 2)``, or neighbours ``(2 i, 2 i + 1)`` when ``interleaved``.

    ``scaling`` stretches the positions for contexts longer than the ones trained
    on by ``"factor"``:

    - ``{"type": "linear", "factor": f}`` divides every frequency by f;
    - ``{"type": "ntk", "factor": f}`` raises the base to
      ``base * f ** (dim / (dim - 2))``: the fastest pair keeps its frequency, the
      slowest has it divided by f;
    - ``{"type": "yarn", "factor": f, "original_length": n}`` keeps the pairs that
      turn more than ``beta_fast`` (32) times in n positions, divides those that
      turn less than ``beta_slow`` (1) times and blends linearly between, and
      multiplies the rotated elements by ``attention_factor`` (0.1 ln f + 1).

    Frequencies are 64-bit and angles are reduced in 64 bits on the device; nothing
    is stored there.  An angle ``p * w`` is off by ``(5 + ln(1 / w)) 2^-53`` of itself
    at most: the rounding of the exponent ``-2 i / dim`` grows by ``ln(1 / w)`` in the
    power, the power, the conversion to turns and the product with the position add
    the rest (a scaling adds its own operations, yarn's blend up to ``factor 2^-53``).
    Positions may be any int64 value; beyond 2^53 they are rounded to 53 bits first,
    so that neighbours may share an angle.
    """

    __slots__ = ("dim", "interleaved", "frequencies", "factor", "_desc")

    def __init__(self, dim: int, *, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[dict] = None):
        if not isinstance(dim, (int, np.integer)) or isinstance(dim, bool):
            raise TypeError(f"Rotary dim must be an int, got {type(dim).__qualname__}")
        if dim < 2 or dim % 2 or dim > 2 * N.ROTARY_PAIRS:
            raise ValueError(f"Rotary dim must be even, 2..{2 * N.ROTARY_PAIRS}, got {dim}")
        base = float(base)
        if not base > 0.0 or not math.isfinite(base):
            raise ValueError(f"Rotary base must be positive and finite, got {base}")
        self.dim = int(dim)
        self.interleaved = bool(interleaved)
        self.frequencies, self.factor = _frequencies(self.dim, base, scaling)
        desc = N.RotaryDesc(dim=self.dim, interleaved=int(self.interleaved), factor=self.factor)
        for i, w in enumerate(self.frequencies):
            desc.turns[i] = w / (2.0 * math.pi)
        self._desc = desc

    def __repr__(self) -> str:
        return f"Rotary({self.dim}, interleaved={self.interleaved})"


_KEYS = {"linear": set(), "ntk": set(),
         "yarn": {"original_length", "beta_fast", "beta_slow", "attention_factor"}}


def _frequencies(dim: int, base: float, scaling: Optional[dict]) -> tuple:
    i = np.arange(dim // 2, dtype=np.float64)
    if scaling is None:
        return base ** (-2.0 * i / dim), 1.0
    kind = scaling.get("type")
    if kind not in _KEYS:
        raise ValueError(f"Rotary scaling type must be one of {sorted(_KEYS)}, got {kind!r}")
    unknown = set(scaling) - _KEYS[kind] - {"type", "factor"}
    if unknown:
        raise ValueError(f"Rotary scaling {kind!r} does not take {sorted(unknown)}")
    factor = float(scaling.get("factor", 0.0))
    if not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError(f"Rotary scaling needs a finite factor of at least 1, got {scaling.get('factor')!r}")
    if kind == "linear":
        return base ** (-2.0 * i / dim) / factor, 1.0
    if kind == "ntk":
        stretched = base * factor ** (dim / (dim - 2)) if dim > 2 else base
        return stretched ** (-2.0 * i / dim), 1.0
    n = float(scaling.get("original_length", 0.0))
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not n > 0.0 or not fast > slow > 0.0 or base == 1.0:
        raise ValueError("Rotary scaling 'yarn' needs an original_length > 0, beta_fast > beta_slow > 0 and a base "
                         "other than 1")

    def pair(turns: float) -> float:  # the pair that turns so often in the original length
        return dim * math.log(n / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
    ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    plain = base ** (-2.0 * i / dim)
    attention = scaling.get("attention_factor")
    attention = 0.1 * math.log(factor) + 1.0 if attention is None else float(attention)
    if not math.isfinite(attention):
        raise ValueError(f"Rotary attention_factor must be finite, got {attention}")
    return plain * (1.0 - ramp) + plain / factor * ramp, attention


__all__ = ["Rotary"]
