"""The batch attention holds what its documentation says: f32 sums, p * vs to 22 bits."""
from __future__ import annotations

import numpy as np
import pytest

from seqbound import few_keys_bound, visible
from seqref import F, Batch, attend, queries
from test_gpu_seq_ops import QK, dev, on_device, ops, torch

pytestmark = pytest.mark.gpu


def spread(b):
    """V scales over a range of 2^12: the 128-column tiles' three-term form."""
    b.vs *= np.exp2(np.floor(b.rng.random(b.vs.shape) * 12) - 6).astype(F)


def run(b, q8, qs, heads, qk, ids=None, n_sel=0):
    pool, seqs = on_device(b)
    out = torch.zeros((b.rows, heads * 128), device="cuda")
    if ids is None:
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=qk)
    else:
        ops.attention_pages(dev(q8), dev(qs), pool, seqs, dev(ids), n_sel, out, qk_scale=qk)
    return out.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("kind", ["few", "wide", "wide_spread", "listed"])
def test_rows_of_few_keys(cuda, kind):
    """Rows of one to four keys, whose error is that of the terms themselves."""
    heads, qk = 16, QK / 64
    wide = kind.startswith("wide")
    lens = [(700, 0)] * 3 if wide else [(4, 0)] * 12 + [(1, i % 4) for i in range(12)]
    b = Batch(lens, 2, 32, seed=len(kind))
    assert (b.rows * heads * b.max_kv > 12 << 20) == wide
    if kind == "wide_spread":
        spread(b)
    q8, qs = queries(b.rng, b.rows, heads)
    ids = np.zeros((b.rows, 2), np.int32) if kind == "listed" else None
    got = run(b, q8, qs, heads, qk, ids, 1)
    want, mag, top = attend(b, q8, qs, heads, qk)
    n = visible(b)
    at = (n >= 1) & (n <= 4)
    assert at.sum() >= 12 and top[at].max() < 0.5
    err, bound = np.abs(got - want)[at], few_keys_bound(mag, top, n[:, None])[at]
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("lens,heads,kv_heads,scales,listed", [
    ([(1, 700), (1, 5), (1, 1300), (1, 95)], 16, 8, "near", 0), ([(2, 3000), (1, 4500)], 16, 8, "near", 0), ([(2, 3000), (1, 4500)], 16, 1, "far", 0),
    ([(420, 4200), (43, 7)], 6, 2, "near", 0), ([(420, 4200), (43, 7)], 6, 2, "far", 0), ([(1, 3000), (240, 51), (33, 900), (9, 0)], 16, 8, "near", 0),
    ([(24, 9000)], 64, 2, "near", 0), ([(24, 9000)], 64, 2, "far", 0), ([(920, 0), (1, 900)], 16, 8, "near", 0),
    ([(7, 3000), (1, 2000)], 16, 8, "near", 40)])
def test_norm_of_the_error(cuda, lens, heads, kv_heads, scales, listed):
    """The whole result is within 1e-6 of float64 (2-norm): some 16 roundings of 2^-24, where a
    key's terms, exponent and weight leave under 4 and f32 sums of up to 1000 keys a wave, with
    partial sums of random signs, about 6.  p * vs as two bf16 numbers leaves 2e-6."""
    b = Batch(lens, kv_heads, 32, seed=len(lens) + heads)
    if scales == "far":
        spread(b)
    q8, qs = queries(b.rng, b.rows, heads)
    ids = np.tile(np.arange(listed, dtype=np.int32) + 3, (b.rows, kv_heads)) if listed else None
    got = run(b, q8, qs, heads, QK / 8, ids, listed)
    want, _, _ = attend(b, q8, qs, heads, QK / 8, True, ids, listed)
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= 1e-6, off
    print("off by", off)
