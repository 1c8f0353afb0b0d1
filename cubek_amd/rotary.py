"""Rotary positions, as ``cache.append`` applies them: the frequencies of a head's pairs and how the pairs lie."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List

from .tensor import TensorHandleRef


@dataclass(frozen=True)
class Rotary:
    """``frequencies``: f32 [n] on the device; the first 2 n entries of a head are turned by position * frequency, entry i with entry
    i + n, or 2 i with 2 i + 1 where ``interleaved``; cosine and sine are multiplied by ``magnitude``."""

    frequencies: TensorHandleRef
    magnitude: float = 1.0
    interleaved: bool = False


def frequencies(turned: int, base: float = 10000.0, factor: float = 1.0) -> List[float]:
    """base^(-2 i / turned) for the pairs of ``turned`` entries; positions ``factor`` times as close for contexts that much longer."""
    if turned < 2 or turned % 2:
        raise ValueError(f"an even number of entries is turned, not {turned}")
    return [base ** (-2.0 * i / turned) / factor for i in range(turned // 2)]


def frequencies_by_parts(turned: int, factor: float, trained: int, base: float = 10000.0, fast: float = 32.0, slow: float = 1.0) -> List[float]:
    """The same for contexts ``factor`` times as long as the ``trained`` one, by parts: pairs that turn more than ``fast`` times within it
    stay, those that turn less than ``slow`` times are slowed down by ``factor``, between them both are mixed linearly in the pair's index.
    The method is "NTK-by-parts" interpolation as YaRN has it (Peng, Quesnelle, Fan, Shippole: YaRN: Efficient Context Window Extension of
    Large Language Models, 2023), with the indexes of both bounds rounded outwards and kept within 0 and ``turned`` - 1."""
    plain = frequencies(turned, base)
    index = lambda turns: turned * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
    low, high = max(0, math.floor(index(fast))), min(turned - 1, math.ceil(index(slow)))
    if high <= 0:  # no pair turns more than ``slow`` times
        return [f / factor for f in plain]
    slowed = lambda i: min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
    return [f * (1.0 - slowed(i)) + f / factor * slowed(i) for i, f in enumerate(plain)]


def magnitude(factor: float) -> float:
    """What cosine and sine are multiplied by beside ``frequencies_by_parts``: 0.1 ln(factor) + 1 (of the same paper)."""
    return 1.0 if factor <= 1.0 else 0.1 * math.log(factor) + 1.0
