"""Rotary frequency tables: the checkpoint's ``rope.inv_freq`` (derived, not in the official
checkpoint) and those of other heads and longer contexts (``rope_frequencies``). They are applied
by :func:`slimdit.ops.rotary`.

ComfyUI's MiniMax-H3 model registers the buffer uninitialised and expects the checkpoint to
carry it. Values: ``1 / 10000 ** (k / 16)`` for k in [0, 16), evaluated entirely in float32
(the reference's slimdit/rope.py:23-27; other spellings round differently in the last ulp).
"""

from __future__ import annotations

import math

import numpy as np

INV_FREQ_LEN = 16
THETA = 10000.0


def rope_inv_freq(length: int = INV_FREQ_LEN, theta: float = THETA) -> np.ndarray:
    """float32 [length]; index 0 is 1.0."""
    k = np.arange(length, dtype=np.float32)
    return np.float32(1.0) / (np.float32(theta) ** (k / np.float32(length)))


def rope_frequencies(rot_dim: int, theta: float = THETA, scaling: str | None = None, factor: float = 1.0,
                     original_length: int | None = None, slow: float = 1.0,
                     fast: float = 32.0) -> tuple[np.ndarray, float]:
    """(float32 [rot_dim/2] frequencies, magnitude) of a head whose first ``rot_dim`` elements rotate:
    theta^(-2j/rot_dim), computed in float64, for contexts ``factor`` times longer than
    ``original_length`` changed by ``scaling``:

    None       unchanged
    "linear"   every frequency divided by factor (position interpolation)
    "ntk"      theta * factor^(rot_dim / (rot_dim - 2)): the slowest frequency is divided by factor,
               the fastest stays
    "parts"    by the turns a frequency makes over original_length: up to ``slow`` turns divided by
               factor, from ``fast`` on unchanged, a linear blend between (NTK by parts)
    "yarn"     "parts", with magnitude 0.1 ln(factor) + 1 (Peng et al., "YaRN", 2023)

    The blend is linear in the turns, as that paper defines it. Checkpoints whose code blends linearly in the
    pair's index between two correction indices were trained with other middle frequencies (the ends agree):
    their own table belongs in ``inv_freq`` then.
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"the rotated part must be a positive even number, got {rot_dim}")
    if not (theta > 0 and factor >= 1.0):
        raise ValueError(f"theta must be positive and factor at least 1, got {theta} and {factor}")
    if scaling not in (None, "linear", "ntk", "parts", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    j = np.arange(rot_dim // 2, dtype=np.float64)
    base = float(theta)
    if scaling == "ntk" and rot_dim > 2:
        base *= factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-2.0 * j / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("parts", "yarn"):
        if original_length is None or original_length < 1 or not slow < fast:
            raise ValueError(f"{scaling} needs original_length and slow < fast")
        keep = np.clip((original_length * freq / (2.0 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    return freq.astype(np.float32), magnitude
