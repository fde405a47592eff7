"""Plain forms of the batch operators over a paged cache, for their tests: numpy
on the host, one f32 operation at a time where the result is bit-exact, float64
where it is not.  A batch is a list of (new rows, keys before them)."""
from __future__ import annotations

import numpy as np

F = np.float32
INV127 = F(1) / F(127)


class Batch:
    """A pool with the batch's pages scattered over it, values everywhere (NaN
    scales in every slot that no sequence's keys fill), tables whose unused
    entries name no page, and row starts with `before` rows in front and `behind`
    rows after the sequences'."""

    def __init__(self, lens, kv_heads, page, seed=0, before=0, behind=0, spare_pages=3, smooth=False):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.kv_heads, self.page = lens, kv_heads, page
        n = [r for r, _ in lens]
        self.start = (before + np.cumsum([0] + n)).astype(np.int32)
        self.rows = int(self.start[-1]) + behind
        self.kv_len = np.array([r + c for r, c in lens], np.int32)
        per = [-(-int(x) // page) for x in np.maximum(self.kv_len, 0)]
        self.n_pages = sum(per) + spare_pages
        order = rng.permutation(self.n_pages)
        self.tables = np.full((len(lens), max(per + [1])), 65535, np.uint16)
        at = 0
        for i, p in enumerate(per):
            self.tables[i, :p] = order[at:at + p]
            at += p
        shape = (self.n_pages, page, kv_heads)
        self.k = rng.integers(-127, 128, shape + (128,)).astype(np.int8)
        if smooth:  # keys of a page near each other
            base = rng.integers(-90, 91, (self.n_pages, 1, kv_heads, 128))
            self.k = np.clip(base + rng.integers(-30, 31, shape + (128,)), -127, 127).astype(np.int8)
        self.v = rng.integers(-127, 128, shape + (128,)).astype(np.int8)
        self.ks = np.full(shape, np.nan, F)
        self.vs = np.full(shape, np.nan, F)
        for i in range(len(lens)):
            t = np.arange(max(int(self.kv_len[i]), 0))
            p = self.tables[i, t // page]
            self.ks[p, t % page] = rng.uniform(0.01, 0.03, (len(t), kv_heads))
            self.vs[p, t % page] = rng.uniform(0.01, 0.03, (len(t), kv_heads))
        self.max_rows = max(n + [0])
        self.max_kv = int(max(list(self.kv_len) + [0]))

    def row_positions(self):
        """(row, sequence, position) of each sequence's rows."""
        return [(int(self.start[s]) + i, s, int(self.kv_len[s]) - r + i)
                for s, (r, _) in enumerate(self.lens) for i in range(r)]

    def keys(self, s, head, tokens):
        """K, V (float64) and which of the tokens lie in a page of the pool."""
        t = np.asarray(tokens)
        p = self.tables[s, t // self.page].astype(np.int64)
        ok = p < self.n_pages
        p = np.where(ok, p, 0)
        at = (p, t % self.page, head)
        with np.errstate(invalid="ignore"):
            k = self.k[at].astype(np.float64) * self.ks[at][..., None].astype(np.float64)
            v = self.v[at].astype(np.float64) * self.vs[at][..., None].astype(np.float64)
        return k, v, ok


def queries(rng, rows, heads):
    return rng.integers(-127, 128, (rows, heads * 128)).astype(np.int8), rng.uniform(0.01, 0.03, (rows, heads)).astype(F)


def attend(b: Batch, q8, qs, heads, scale, causal=True, ids=None, n_sel=0):
    """float64 attention [rows][heads * 128], the softmax-weighted |v| and the
    largest |score| of each (row, head): what an error bound is relative to."""
    g = heads // b.kv_heads
    out = np.zeros((b.rows, heads, 128))
    mag = np.zeros((b.rows, heads, 128))
    top = np.zeros((b.rows, heads))
    if ids is None:  # a sequence's rows and a KV head's query heads at once
        for s, (n, _) in enumerate(b.lens):
            r0, kv = int(b.start[s]), max(int(b.kv_len[s]), 0)
            if n == 0 or kv == 0:
                continue
            pos = int(b.kv_len[s]) - n + np.arange(n)
            for kvh in range(b.kv_heads):
                k, v, ok = b.keys(s, kvh, np.arange(kv))
                k[~ok], v[~ok] = 0, 0
                sees = ok[None] & ((np.arange(kv)[None] <= pos[:, None]) if causal else True)
                any_ = sees.any(1)
                vsum = sees @ (np.abs(v) + 128)
                for h in range(kvh * g, kvh * g + g):
                    q = q8[r0:r0 + n, h * 128:(h + 1) * 128].astype(np.float64) * qs[r0:r0 + n, h, None].astype(np.float64)
                    x = np.where(sees, (q @ k.T) * float(F(scale)), -np.inf)
                    p = np.exp(x - np.where(any_, x.max(1), 0)[:, None])
                    p /= np.maximum(p.sum(1), 1e-300)[:, None]
                    out[r0:r0 + n, h], mag[r0:r0 + n, h] = p @ v, p @ np.abs(v) + 2.0 ** -109 * vsum
                    top[r0:r0 + n, h] = np.where(any_, np.abs(np.where(sees, x, 0)).max(1), 0)
        return out.reshape(b.rows, -1), mag.reshape(b.rows, -1), np.repeat(top, 128, 1)
    for row, s, pos in b.row_positions():  # listed pages, row by row
        visible = pos + 1
        for kvh in range(b.kv_heads):
            pages = [p for p in ids[row, kvh * n_sel:(kvh + 1) * n_sel] if 0 <= p < b.tables.shape[1]]
            tok = np.concatenate([np.arange(p * b.page, (p + 1) * b.page) for p in pages] or [np.zeros(0, int)]).astype(int)
            tok = tok[tok < visible]
            k, v, ok = b.keys(s, kvh, tok)
            k, v = k[ok], v[ok]
            if len(k) == 0:
                continue
            for h in range(kvh * g, kvh * g + g):
                q = q8[row, h * 128:(h + 1) * 128].astype(np.float64) * float(qs[row, h])
                x = (k @ q) * float(F(scale))
                p = np.exp(x - x.max())
                p /= p.sum()
                out[row, h], top[row, h] = p @ v, np.abs(x).max()
                mag[row, h] = p @ np.abs(v) + 2.0 ** -109 * (np.abs(v) + 128).sum(0)
    return out.reshape(b.rows, -1), mag.reshape(b.rows, -1), np.repeat(top, 128, 1)


def attend_bound(mag, top, n_keys):
    """How far a correct f32 result may be from float64.  A score takes three f32
    roundings and its base-2 exponent two more: 5 * 2^-24 |x| absolute, i.e.
    relative in p, for p and for the maximum's term; exp2 and the weight's two
    products 2^-22; P as a sum of two bf16 numbers 2^-17 (half a step of the second,
    2^-9 of a remainder of 2^-9, twice: numerator only, rounded up); the numerator's
    and denominator's sums of n terms 2 n 2^-24; all relative to sum p |v|.  A weight
    below the smallest normal float, relative to the largest weight of 1, may come
    out as 0, and so may its product with a V scale: 2^-126 (|v| + 128) a key, which
    attend adds to the magnitudes as 2^17 times that."""
    return mag * (2.0 ** -17 + 2.0 ** -22 + 10 * top * 2.0 ** -24 + 2 * n_keys * 2.0 ** -24) + 1e-30


def quantise(x):
    """Per-head int8 of f32 [rows][heads * 128]: (q8, scales)."""
    x = x.reshape(len(x), -1, 128)
    scale = (np.abs(x).max(-1) * INV127).astype(F)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = (x / scale[..., None]).astype(F)
    q = np.clip(np.rint(np.nan_to_num(q, nan=0.0, posinf=127.0, neginf=-127.0)), -127, 127).astype(np.int8)
    return q.reshape(len(x), -1), scale


def head_norm(x, w):
    """Per-head RMSNorm of f32 [...][128] in the framework's order of additions."""
    q = (x * x).reshape(*x.shape[:-1], 4, 32)
    while q.shape[-1] > 1:
        q = (q[..., 0::2] + q[..., 1::2]).astype(F)
    q = q[..., 0]
    ss = (((q[..., 0] + q[..., 1]) + q[..., 2]) + q[..., 3]).astype(F) * F(1 / 128) + F(1e-6)
    r = F(1) / np.sqrt(ss).astype(F)
    return ((x * r[..., None]).astype(F) * w).astype(F)


def rotate(x, cos, sin, rot, interleaved):
    """x f32 [heads][128] at one position (cos, sin [rot / 2])."""
    y = x.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        y[:, a] = x[:, a] * cos[i] - x[:, b] * sin[i]
        y[:, b] = x[:, a] * sin[i] + x[:, b] * cos[i]
    return y


def bounds_of(k8, ks):
    """Bounds row [256] and scale of one page's keys int8 [tokens][128], f32 [tokens]."""
    x = k8.astype(F) * ks[:, None]
    lo, hi = x.min(0), x.max(0)
    scale = F(max(np.abs(lo).max(), np.abs(hi).max())) * INV127
    if scale == 0:
        return np.zeros(256, np.int8), F(0)
    q = np.concatenate((np.floor((lo / scale).astype(F)), np.ceil((hi / scale).astype(F))))
    return np.clip(q, -127, 127).astype(np.int8), scale


def select(b: Batch, q8, qs, heads, bounds, bscale, n_sel):
    """ids int32 [rows][kv_heads * n_sel]; rows of no sequence keep -9."""
    g = heads // b.kv_heads
    ids = np.full((b.rows, b.kv_heads, n_sel), -9, np.int32)
    for row, s, pos in b.row_positions():
        ids[row] = -1
        if pos < 0:
            continue
        last = pos // b.page
        pages = b.tables[s, :last + 1].astype(np.int64)
        for kvh in range(b.kv_heads):
            score = np.full(last + 1, -np.inf, F)
            for i, p in enumerate(pages):
                if p >= b.n_pages:
                    continue
                lo, hi = bounds[p * b.kv_heads + kvh, :128].astype(np.int64), bounds[p * b.kv_heads + kvh, 128:].astype(np.int64)
                for h in range(kvh * g, kvh * g + g):
                    q = q8[row, h * 128:(h + 1) * 128].astype(np.int64)
                    x = F(F(F(int((q * np.where(q > 0, hi, lo)).sum())) * bscale[p, kvh]) * qs[row, h])
                    score[i] = np.inf if x != x else max(score[i], x)
            score[last] = np.inf
            if np.isposinf(score[:last]).any():
                raise ValueError("an infinite score ties with the row's own page")
            pick = np.sort(np.argsort(-score, kind="stable")[:n_sel])
            ids[row, kvh, :len(pick)] = pick
    return ids.reshape(b.rows, -1)
