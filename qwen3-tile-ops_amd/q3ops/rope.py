"""Rotary position tables for ops.rope_append_paged (and the model's cos/sin rows).

Angles are computed in float64 and rounded once to float32, as
tools/convert_pqwf.py:46-52 does for the plain tables; the context-extension
scalings are position interpolation (linear), NTK-aware base scaling (ntk) and
YaRN's interpolation by parts with its attention factor (yarn).
"""
from __future__ import annotations

import math

import numpy as np

__all__ = ["rope_tables"]


def _yarn_ramp(half: int, theta: float, original: int, beta_fast: float, beta_slow: float) -> np.ndarray:
    """YaRN's ramp: 1 where a dimension turns more than beta_fast times over the original
    context (left as it is), 0 where less than beta_slow times (interpolated),
    linear in the dimension's index between."""
    def dim(turns: float) -> float:
        return half * math.log(original / (turns * 2.0 * math.pi)) / math.log(theta)

    lo, hi = math.floor(dim(beta_fast)), math.ceil(dim(beta_slow))
    lo, hi = max(lo, 0), min(hi, 2 * half - 1)
    return 1.0 - np.clip((np.arange(half) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)


def rope_tables(positions: int, rot_dim: int = 128, theta: float = 1e6, scaling: str | None = None,
                factor: float = 1.0, original: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                attention_factor: float | None = None) -> tuple[np.ndarray, np.ndarray]:
    """cos, sin float32 [positions, rot_dim / 2] of the angles p * f_i,
    f_i = theta^(-2 i / rot_dim).

    scaling None: as they are.  "linear": positions divided by factor.  "ntk":
    theta raised to theta * factor^(rot_dim / (rot_dim - 2)), so that the slowest
    dimension is slowed by factor and the fastest not at all.  "yarn": dimensions
    that turn often over the original context are left, slow ones divided by
    factor, those between blended, and cos and sin multiplied by
    attention_factor (0.1 ln factor + 1 if not given)."""
    if rot_dim <= 0 or rot_dim > 128 or rot_dim % 2:
        raise ValueError("rot_dim is even, from 2 to 128")
    if positions < 0 or not 0 < theta < math.inf or not 1.0 <= factor < math.inf:
        raise ValueError("positions >= 0, theta > 0 and factor >= 1, both finite")
    half = rot_dim // 2
    i = np.arange(half, dtype=np.float64)
    scale = 1.0
    if scaling == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs rot_dim > 2")
        theta = theta * factor ** (rot_dim / (rot_dim - 2))
    f = theta ** (-i / half)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if original <= 0 or theta <= 1.0 or not 0 < beta_slow <= beta_fast < math.inf:
            raise ValueError("yarn scaling needs the original context length, theta > 1 and beta_fast >= beta_slow > 0")
        if attention_factor is not None and not math.isfinite(attention_factor):
            raise ValueError("attention_factor must be finite")
        keep = _yarn_ramp(half, theta, original, beta_fast, beta_slow)
        f = f * keep + f / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0 if attention_factor is None else attention_factor
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    a = np.arange(positions, dtype=np.float64)[:, None] * f
    return (np.cos(a) * scale).astype(np.float32), (np.sin(a) * scale).astype(np.float32)
