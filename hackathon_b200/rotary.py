"""Rotary frequencies as phase steps, the form the rotary kernels take.

The kernels turn pair i of a head at position p by ``p * step_i / 2**64`` turns, the product taken
modulo 2**64: a step is the fraction of a turn one position adds, in 64-bit fixed point.  A far
position loses nothing to range reduction, and no table of sines is read.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np


def rotary_frequencies(rotary_dim: int, base: float = 10000.0) -> np.ndarray:
    """Radians a position of each pair: ``base ** (-2 i / rotary_dim)``, float64 [rotary_dim / 2]."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if not base > 0:
        raise ValueError("base must be positive")
    return float(base) ** (-np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)


def phase_steps(frequencies) -> np.ndarray:
    """Radians a position -> the kernels' int64 phase steps (turns times 2**64, modulo one turn)."""
    f = np.asarray(frequencies, dtype=np.float64)
    if f.ndim != 1 or not np.all(np.isfinite(f)):
        raise ValueError("frequencies must be a finite vector")
    steps = [int(math.ldexp(v / (2.0 * math.pi), 64)) & 0xFFFFFFFFFFFFFFFF for v in f.tolist()]
    return np.array(steps, dtype=np.uint64).view(np.int64)


def rotary_steps(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 ) -> Tuple[np.ndarray, float]:
    """Phase steps int64 [rotary_dim / 2] and the ``scale`` on sines and cosines.

    ``scaling`` stretches a model trained on ``original_length`` positions by ``factor``:

    * ``None``: as trained;
    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: the base raised to ``base * factor ** (d / (d - 2))``, d = ``rotary_dim``, so that the slowest
      pair is slowed by ``factor`` and the fastest is left alone;
    * ``"turns"``: pairs that make more than ``beta_fast`` turns within ``original_length`` stay, those that make
      fewer than ``beta_slow`` are slowed by ``factor``, a linear ramp in turns between; sines and cosines are
      multiplied by ``0.1 ln(factor) + 1``.
    """
    if not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    scale = 1.0
    f = rotary_frequencies(rotary_dim, base)
    if scaling == "linear":
        f = f / factor
    elif scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling the base needs more than one pair")
        f = rotary_frequencies(rotary_dim, base * factor ** (rotary_dim / (rotary_dim - 2)))
    elif scaling == "turns":
        if not beta_fast > beta_slow:
            raise ValueError("beta_fast must be above beta_slow")
        turns = original_length * f / (2.0 * math.pi)
        keep = np.clip((turns - beta_slow) / (beta_fast - beta_slow), 0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling is not None:
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'base' or 'turns'")
    return phase_steps(f), scale
