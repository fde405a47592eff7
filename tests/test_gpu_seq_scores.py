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


def positive(kind, seed):
    """Queries, keys and their scales above zero: a key's score has its scale's sign."""
    b = Batch(KINDS[kind], 2, 32, seed=seed)
    heads = 16 if kind == "many" else 4
    b.k[:] = b.rng.integers(1, 128, b.k.shape)
    q8, qs = queries(b.rng, b.rows, heads)
    return b, heads, np.maximum(np.abs(q8), 1).astype(np.int8), qs


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low", [-np.inf, -3e38])
def test_scores_of_minus_infinity(cuda, kind, low):
    """Keys whose scores are -inf (by their scale, or past the floats' range) have no
    weight: rows that see none but such get zeros, the others what the other keys give."""
    b, heads, q8, qs = positive(kind, 5)
    n_sel = 20
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    hidden = b.tables.copy()
    for s, pages in ((0, range(15)), (1, range(2)), (2, range(1))):  # sequence 1: all its keys
        for i in pages:
            if i * 32 < b.kv_len[s]:
                n = min(32, b.kv_len[s] - i * 32)
                b.ks[b.tables[s, i], :n] = low
                hidden[s, i] = 65535
    got = run(kind, b, q8, qs, heads, ids, n_sel)
    b.tables = hidden  # the same as pages outside the pool
    want, mag, top = attend(b, q8, qs, heads, QK, True, ids if kind == "listed" else None, n_sel)
    assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:4].tolist()
    assert (np.abs(got - want) <= attend_bound(mag, top, b.max_kv)).all()
    assert (got[int(b.start[1]):int(b.start[2])] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_scores_of_infinity(cuda, kind):
    """A key whose score is inf makes the rows that see it NaN, whole rows of a head, and
    no other; so does an infinite V scale."""
    b, heads, q8, qs = positive(kind, 6)
    n_sel = 4
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    plain = run(kind, b, q8, qs, heads, ids, n_sel)
    assert np.isfinite(plain).all()
    _, mag, top = attend(b, q8, qs, heads, QK, True, ids if kind == "listed" else None, n_sel)
    twice = 2 * attend_bound(mag, top, b.max_kv)
    for name in ("ks", "vs"):
        t = 33  # of sequence 0, KV head 1: the heads of the upper half
        at = b.tables[0, t // 32], t % 32, 1
        keep = getattr(b, name)[at]
        getattr(b, name)[at] = np.inf
        got, want = run(kind, b, q8, qs, heads, ids, n_sel), plain.copy()
        getattr(b, name)[at] = keep
        sees = [r for r, s, p in b.row_positions() if s == 0 and p >= t]
        want[sees, heads * 64:] = np.nan
        same = np.isnan(got) == np.isnan(want)
        assert same.all(), (name, np.argwhere(~same)[:4].tolist())
        assert (np.abs(got - want) <= twice)[~np.isnan(want)].all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 24, 2.0 ** 27, 2.0 ** 32, 2.0 ** 60])
def test_huge_scores(cuda, kind, size):
    """Scores of millions and more: one key has all the weight of a row where the next
    largest score lies further below than f32 roundings of both can move them."""
    b, heads, q8, qs = positive(kind, 7)
    b.ks *= F(size)
    n_sel = 20
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    got = run(kind, b, q8, qs, heads, ids, n_sel).reshape(b.rows, heads, 128)
    assert np.isfinite(got).all()
    checked = 0
    for row, s, pos in b.row_positions():
        for h in range(heads):
            k, v, _ = b.keys(s, h // (heads // 2), np.arange(min(pos + 1, n_sel * 32) if kind == "listed" else pos + 1))
            x = (k @ q8[row, h * 128:(h + 1) * 128].astype(np.float64)) * float(qs[row, h]) * QK
            first = int(np.argmax(x))
            # a score and its distance from the largest: ten roundings of 2^-24 each; e^-30 is none of the weight
            if len(x) > 1 and x[first] - np.partition(x, -2)[-2] < 20 * 2.0 ** -24 * x[first] + 30:
                continue
            checked += 1
            # the weight's products, P's terms (2^-22 each) and the division; 1100 other keys
            # at most, of e^-30 and 127 * 0.03
            assert (np.abs(got[row, h] - v[first]) <= 2.0 ** -20 * np.abs(v[first]) + 4e-10).all(), (row, h)
    assert checked > b.rows * heads // 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low", [-1e4, -1e10, -1e20, -1e30])
def test_scores_far_below_the_others(cuda, kind, low):
    """Keys pushed far down by their scale, whole blocks of them in front of the others and
    single ones between: the rest comes out as without them."""
    b, heads, q8, qs = positive(kind, 8)
    n_sel = 20
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    hidden = b.tables.copy()
    for i in (0, 1, 2, 3, 4, 6, 9):
        b.ks[b.tables[0, i]] = low
        hidden[0, i] = 65535
    got = run(kind, b, q8, qs, heads, ids, n_sel)
    b.tables = hidden  # the same as pages outside the pool: weights below 2^-1000
    want, mag, top = attend(b, q8, qs, heads, QK, True, ids if kind == "listed" else None, n_sel)
    sees = [r for r, s, p in b.row_positions() if s or p >= 5 * 32]
    assert (np.abs(got - want) <= attend_bound(mag, top, b.max_kv))[sees].all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1.0, 2.0 ** 4, 2.0 ** 30, 2.0 ** 60])
def test_equal_scores(cuda, kind, size):
    """One key over and over: all have the same weight, however large their score."""
    b, heads, q8, qs = positive(kind, 9)
    b.k[:] = b.k[0, 0]
    b.ks[:] = np.where(np.isnan(b.ks), np.nan, F(0.0217) * F(size))
    n_sel = 20
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    got = run(kind, b, q8, qs, heads, ids, n_sel)
    b.ks[:] = np.where(np.isnan(b.ks), np.nan, 0)  # scores of no size: weights of 1
    want, mag, _ = attend(b, q8, qs, heads, QK, True, ids if kind == "listed" else None, n_sel)
    assert (np.abs(got - want) <= attend_bound(mag, 0, b.max_kv)).all()
