"""The batch attention where scores and V scales are far apart, infinite or huge."""
from __future__ import annotations

import numpy as np
import pytest

from seqref import F, Batch, attend, attend_bound, quantise, queries
from test_gpu_seq_ops import QK, dev, on_device, ops, torch

pytestmark = pytest.mark.gpu

# 16-column tiles, 128-column ones (more than 12 << 20 (row, head, key) triples), listed pages
KINDS = {"few": [(5, 700), (1, 40), (3, 2)], "many": [(800, 300), (1, 40), (100, 700)], "listed": [(5, 700), (1, 40), (3, 2)]}


def run(kind, b, q8, qs, heads, ids=None, n_sel=0, qk=QK):
    assert (b.rows * heads * b.max_kv > 12 << 20) == (kind == "many")
    pool, seqs = on_device(b)
    out = torch.empty((b.rows, heads * 128), device="cuda")
    o8, os_ = torch.empty((b.rows, heads * 128), dtype=torch.int8, device="cuda"), torch.empty((b.rows, heads), device="cuda")
    for kw in ({"out": out}, {"o8": o8, "os": os_}):
        if kind == "listed":
            ops.attention_pages(dev(q8), dev(qs), pool, seqs, dev(ids), n_sel, qk_scale=qk, **kw)
        else:
            ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, qk_scale=qk, **kw)
    got = out.cpu().numpy()
    r8, rs = quantise(got)
    fine = np.isfinite(rs)
    assert np.array_equal(os_.cpu().numpy()[fine], rs[fine])
    assert np.array_equal(o8.cpu().numpy().reshape(*rs.shape, 128)[fine], r8.reshape(*rs.shape, 128)[fine])
    return got


@pytest.mark.parametrize("kind", ["few", "many"])
@pytest.mark.parametrize("margin", [20, 30, 40])
def test_zero_values_under_the_largest_score(cuda, kind, margin):
    """The first key (an attention sink) has an all-zero V row, whose scale is 0, and a
    score `margin` above the others' in base 2: the result is the others', small as they are."""
    heads, qk = 16, float(F(128 ** -0.5))
    b = Batch(KINDS[kind], 2, 32, seed=margin)
    b.k[:] = np.clip(b.k, -30, 30)
    q8 = b.rng.integers(40, 128, (b.rows, heads * 128)).astype(np.int8)
    qs = np.full((b.rows, heads), 0.02, F)
    # q . 127 is 127 * 83.5 * 128 on average
    for s in range(len(b.lens)):
        at = int(b.tables[s, 0]), 0
        b.k[at], b.ks[at] = 127, margin / (127 * 83.5 * 128 * 0.02 * qk * np.log2(np.e))
        b.v[at], b.vs[at] = 0, 0
    got = run(kind, b, q8, qs, heads, qk=qk)
    want, mag, top = attend(b, q8, qs, heads, qk)
    err, bound = np.abs(got - want), attend_bound(mag, top, b.max_kv)
    assert (err <= bound).all(), float((err / bound).max())
