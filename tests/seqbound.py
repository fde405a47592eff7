"""What the batch attention's documented precision allows, for rows of few keys, where no
long sum hides it."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # one f32 rounding, relative


def few_keys_bound(mag, top, n):
    """How far rows of n visible keys (an array like mag) may be from float64, relative to
    mag = sum p |v| / sum p, for n of one 32-key block and scores |x| <= top well below 1.

    A score takes five f32 roundings (two scales, qk_scale, log2 e and its own value), its
    distance from the maximum's one more of twice the size: 7 U top in the exponent, under
    12 U top with the maximum's own, in the numerator and in the denominator: 24 U top.
    exp2 is off by one step of 2^-23, in both: 4 U.  p * vs: U; as three bf16 numbers U at
    most, as two f16 numbers 2^-22 (p vs lies within 2^8 of the largest): 4 U.  Each of up to three
    partial products a key is added with a rounding that may cut: 2 U.  The denominator's sum: U
    a key.  A division, or a reciprocal and a product: 2 U.  No key is in another wave or
    split, so no factor joins them."""
    return mag * U * (24 * top + 4 + 1 + 4 + 6 * n + n + 2) + 1e-30


def visible(b, causal=True):
    """How many keys each row of a Batch sees [rows]; 0 for rows of no sequence."""
    n = np.zeros(b.rows, int)
    for row, s, pos in b.row_positions():
        n[row] = max(pos + 1, 0) if causal else max(int(b.kv_len[s]), 0)
    return n


def as_bf16_terms(x, terms):
    """float32 x as the sum of that many bf16 numbers (round to nearest, ties to even)."""
    rest, total = x.astype(np.float32), np.zeros(x.shape)
    for _ in range(terms):
        i = rest.view(np.uint32).astype(np.uint64)
        t = (((i + 0x7FFF + ((i >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)
        total += t
        rest = rest - t
    return total


def as_f16_terms(x, terms):
    rest, total = x.astype(np.float32), np.zeros(x.shape)
    for _ in range(terms):
        t = rest.astype(np.float16).astype(np.float32)
        total += t
        rest = rest - t
    return total
