"""The bounds that the batch attention's precision is tested with tell its terms apart:
products p * vs held to fewer bits than documented lie outside, on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

from seqbound import as_bf16_terms, as_f16_terms, few_keys_bound
from seqref import F


def rows_of(n, count, seed):
    """count rows of n keys: p vs (f32, the largest in f16's upper range), V, sum p, and
    the weighted |V|."""
    rng = np.random.default_rng(seed)
    p = np.exp(rng.uniform(-0.2, 0.2, (count, n))).astype(F)
    p /= p.max(1, keepdims=True)
    vs = rng.uniform(0.01, 0.03, (count, n)).astype(F)
    pv = (p * vs * F(2.0 ** 15)).astype(F)
    v = rng.integers(-127, 128, (count, n, 128)).astype(np.float64)
    return pv, v, p.astype(np.float64).sum(1) * 2.0 ** 15


@pytest.mark.parametrize("n", [1, 2, 4])
def test_fewer_terms_are_seen(n):
    pv, v, total = rows_of(n, 200, n)
    times = lambda w: (w.astype(np.float64)[..., None] * v).sum(1) / total[:, None]  # noqa: E731
    want, mag = times(pv), (pv.astype(np.float64)[..., None] * np.abs(v)).sum(1) / total[:, None]
    bound = few_keys_bound(mag, 0.2, n)
    over = lambda w: (np.abs(times(w) - want) > bound).mean()  # noqa: E731
    assert over(as_bf16_terms(pv, 3)) == 0 and over(as_f16_terms(pv, 2)) == 0
    assert over(as_bf16_terms(pv, 2)) > 0.05 and over(as_bf16_terms(pv, 1)) > 0.5 and over(as_f16_terms(pv, 1)) > 0.5


def test_fewer_terms_are_seen_in_the_norm():
    pv, v, total = rows_of(700, 40, 9)
    times = lambda w: (w.astype(np.float64)[..., None] * v).sum(1) / total[:, None]  # noqa: E731
    want = times(pv)
    off = lambda w: np.linalg.norm(times(w) - want) / np.linalg.norm(want)  # noqa: E731
    assert off(as_bf16_terms(pv, 3)) < 1e-7 and off(as_f16_terms(pv, 2)) < 3e-7
    assert off(as_bf16_terms(pv, 2)) > 1.5e-6 and off(as_f16_terms(pv, 1)) > 1e-4
