"""The batch operators over one paged cache against their plain forms."""
from __future__ import annotations

import numpy as np
import pytest

import seqref
from conftest import bits_equal, describe_diff
from seqref import F, Batch, attend, attend_bound, quantise, queries

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from q3ops import ops  # noqa: E402
from q3ops.rope import rope_tables  # noqa: E402

QK = float(F(128 ** -0.5))


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def on_device(b: Batch, max_rows=None, max_kv=None):
    kv = b.kv_heads
    pool = ops.kv_pool(dev(b.k.reshape(b.n_pages, b.page, kv * 128)), dev(b.v.reshape(b.n_pages, b.page, kv * 128)),
                       dev(b.ks), dev(b.vs))
    seqs = ops.sequences(pool, dev(b.tables), dev(b.start), dev(b.kv_len), b.max_rows if max_rows is None else max_rows,
                         b.max_kv if max_kv is None else max_kv)
    return pool, seqs


def check_attention(b, heads, causal=True, ids=None, n_sel=0, seed=1):
    rng = np.random.default_rng(seed)
    q8, qs = queries(rng, b.rows, heads)
    pool, seqs = on_device(b)
    tq, ts = dev(q8), dev(qs)
    out = torch.full((b.rows, heads * 128), 7.5, device="cuda")
    o8 = torch.full((b.rows, heads * 128), 99, dtype=torch.int8, device="cuda")
    os_ = torch.full((b.rows, heads), 7.5, device="cuda")
    if ids is None:
        call = lambda **kw: ops.attention_varlen_paged(tq, ts, pool, seqs, causal=causal, qk_scale=QK, **kw)  # noqa: E731
    else:
        ti = dev(ids)
        call = lambda **kw: ops.attention_pages(tq, ts, pool, seqs, ti, n_sel, qk_scale=QK, **kw)  # noqa: E731
    call(out=out)
    call(o8=o8, os=os_)
    got = out.cpu().numpy()
    want, mag, top = attend(b, q8, qs, heads, QK, causal, ids, n_sel)
    mine = np.zeros(b.rows, bool)
    mine[[r for r, _, _ in b.row_positions()]] = True
    assert (got[~mine] == 7.5).all() and (o8.cpu().numpy()[~mine] == 99).all() and (os_.cpu().numpy()[~mine] == 7.5).all()
    err, bound = np.abs(got - want)[mine], attend_bound(mag, top, max(b.max_kv, n_sel * b.page))[mine]
    assert np.isfinite(got).all()
    assert (err <= bound).all(), (float((err / bound).max()), np.argwhere(err > bound)[:4].tolist())
    r8, rs = quantise(got[mine])  # the int8 form rounds the f32 form's values
    assert bits_equal(os_.cpu().numpy()[mine], rs), describe_diff(os_.cpu().numpy()[mine], rs)
    assert bits_equal(o8.cpu().numpy()[mine], r8), describe_diff(o8.cpu().numpy()[mine], r8)
    again = torch.empty_like(out)
    call(out=again)
    assert torch.equal(again[dev(mine)], out[dev(mine)])


LENS = {
    "one": [(1, 0)],
    "two_keys": [(1, 1)],
    "page_edges": [(1, 31), (1, 32), (1, 33), (1, 63), (1, 64)],
    "decode": [(1, 700), (1, 5), (1, 1300), (1, 95), (1, 0)],
    "prompt": [(97, 0)],
    "chunks": [(3, 40), (33, 100), (64, 64), (130, 17)],
    "empty_ones": [(0, 50), (1, 20), (0, 0), (5, 3), (0, 9)],
    "none_before": [(4, -2), (3, -3), (2, 10), (40, -38)],  # rows at negative positions see nothing
    "long": [(2, 3000), (1, 4500)],
}


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,kv_heads,page", [(16, 8, 32), (6, 2, 96)])
def test_attention(cuda, lens, heads, kv_heads, page):
    check_attention(Batch(LENS[lens], kv_heads, page, seed=len(lens)), heads)


@pytest.mark.parametrize("heads,kv_heads,page", [(8, 8, 64), (20, 4, 32), (16, 1, 128), (33, 1, 32), (64, 2, 256), (24, 2, 32)])
@pytest.mark.parametrize("lens", ["decode", "chunks"])
def test_attention_head_layouts(cuda, heads, kv_heads, page, lens):
    check_attention(Batch(LENS[lens], kv_heads, page, seed=heads), heads)


@pytest.mark.parametrize("lens", ["decode", "chunks", "empty_ones", "none_before", "prompt"])
def test_attention_not_causal(cuda, lens):
    check_attention(Batch(LENS[lens], 4, 32, seed=5), 8, causal=False)


# more than 12 << 20 (row, head, key) triples: the 128-column tiles, beside 16-column
# ones for the sequences of few rows
WIDE = {
    "prompt": ([(920, 0), (1, 900)], 16, 8, 32),
    "chunk": ([(860, 101)], 16, 8, 128),
    "mixed": ([(1, 3000), (240, 51), (0, 5), (33, 900), (2, 40), (9, 0)], 16, 8, 32),
    "group_of_three": ([(420, 4200), (43, 7)], 6, 2, 96),
    "one_kv_head": ([(200, 4000), (1, 64)], 16, 1, 32),
    "group_of_33": ([(100, 4000)], 33, 1, 64),
    "negative_positions": ([(200, -150), (64, 6400), (40, -40)], 16, 2, 32),
    "many_splits": ([(24, 9000)], 64, 2, 256),
    "no_groups": ([(700, 500), (17, 33)], 16, 16, 32),
}


@pytest.mark.parametrize("name", WIDE)
def test_attention_wide(cuda, name):
    lens, heads, kv_heads, page = WIDE[name]
    b = Batch(lens, kv_heads, page, seed=len(name), before=1, behind=2)
    assert b.rows * heads * b.max_kv > 12 << 20
    check_attention(b, heads)


@pytest.mark.parametrize("name", ["mixed", "negative_positions", "many_splits"])
def test_attention_wide_not_causal(cuda, name):
    lens, heads, kv_heads, page = WIDE[name]
    check_attention(Batch(lens, kv_heads, page, seed=8), heads, causal=False)


def test_attention_wide_bad_pages(cuda):
    b = Batch([(340, 500), (250, 1000), (60, 1000)], 2, 32, seed=1)
    b.tables[0, [0, 3, 24]] = [b.n_pages, 65535, b.n_pages + 7]
    b.tables[1, 4:30] = 65535
    b.tables[2] = 65535
    assert b.rows * 16 * b.max_kv > 12 << 20
    check_attention(b, 16)


@pytest.mark.parametrize("what", ["wide", "within", "zeros", "tiny", "huge", "negative", "queries"])
def test_attention_wide_scales(cuda, what):
    """V scales both sides of what the f16 terms take: a range of 2^8 and more, one of 2^7, zeros,
    near either end of the floats, negative; query scales of zero and below."""
    b = Batch([(800, 300), (1, 40), (100, 700)], 2, 32, seed=3)
    assert b.rows * 16 * b.max_kv > 12 << 20
    scale = {"wide": lambda u: np.exp2(np.floor(u * 9) - 4), "within": lambda u: np.exp2(np.floor(u * 7) - 3),
             "zeros": lambda u: np.where(u < 0.3, 0, 1), "tiny": lambda u: np.full_like(u, 2.0 ** -90),
             "huge": lambda u: np.full_like(u, 2.0 ** 90), "negative": lambda u: np.where(u < 0.5, -1, 1), "queries": np.ones_like}[what]
    b.vs *= scale(b.rng.random(b.vs.shape)).astype(F)
    q8, qs = queries(b.rng, b.rows, 16)
    if what == "queries":
        qs[::3] = 0
        qs[1::3] *= -1
        qs[2::9, ::3] *= -1
    want, mag, top = attend(b, q8, qs, 16, QK)
    pool, seqs = on_device(b)
    out = torch.empty((b.rows, 2048), device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
    got = out.cpu().numpy()
    err, bound = np.abs(got - want), attend_bound(mag, top, b.max_kv)
    assert np.isfinite(got).all() and (err <= bound).all(), float((err / bound).max())


def test_attention_wide_strided(cuda):
    """Result rows that 16-byte words do not fit."""
    b = Batch([(800, 300), (1, 40)], 2, 32, seed=3)
    q8, qs = queries(b.rng, b.rows, 16)
    want, mag, top = attend(b, q8, qs, 16, QK)
    pool, seqs = on_device(b)
    wo = torch.full((b.rows, 2048 + 7), 7.5, device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, wo[:, 3:2051], qk_scale=QK)
    got = wo.cpu().numpy()
    assert (np.abs(got[:, 3:2051] - want) <= attend_bound(mag, top, b.max_kv)).all()
    assert (got[:, :3] == 7.5).all() and (got[:, 2051:] == 7.5).all()


def test_attention_wide_bad_lengths(cuda):
    b = Batch([(300, 1300), (300, 500)], 2, 32, behind=4)
    assert b.rows * 16 * b.max_kv > 12 << 20
    q8, qs = queries(b.rng, b.rows, 16)
    want, mag, top = attend(b, q8, qs, 16, QK)
    pool, _ = on_device(b)
    kv_len = b.kv_len.copy()
    for wrong in (1 << 30, 2147483647, -5, -2147483648):
        kv_len[0] = wrong
        seqs = ops.sequences(pool, dev(b.tables), dev(b.start), dev(kv_len), b.max_rows, b.max_kv)
        out = torch.full((b.rows, 2048), 7.5, device="cuda")
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
        got = out.cpu().numpy()
        assert (np.abs(got - want) <= attend_bound(mag, top, b.max_kv))[300:600].all() and (got[600:] == 7.5).all()
    for start in ([0, 300, 1 << 30], [-7, 300, 600], [-2147483648, 2147483647, 600], [600, 300, 0]):
        seqs = ops.sequences(pool, dev(b.tables), dev(np.array(start, np.int32)), dev(b.kv_len), b.max_rows, b.max_kv)
        out = torch.full((b.rows + 8, 2048), 7.5, device="cuda")
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
        assert (out.cpu().numpy()[b.rows:] == 7.5).all()


def test_attention_rows_around_the_sequences(cuda):
    check_attention(Batch([(3, 100), (1, 50), (40, 8)], 8, 32, before=5, behind=9), 16)
    check_attention(Batch([(1, 100), (1, 50)], 8, 32, before=2, behind=3), 16)


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_bad_pages(cuda, rows):
    """A page id outside the pool hides its keys, whichever it is."""
    b = Batch([(rows, 500), (rows, 300)], 2, 32, seed=rows)
    b.tables[0, [0, 3, 9]] = [b.n_pages, 65535, b.n_pages + 7]
    b.tables[1, :4] = 65535
    check_attention(b, 4)


def test_attention_every_page_bad(cuda):
    b = Batch([(1, 200), (40, 200)], 2, 32)
    b.tables[:] = 65535
    check_attention(b, 4)


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_bad_lengths(cuda, rows):
    """Lengths and starts that no caller should hand over stay in bounds: every
    row of the sequences that are right is right, nothing else is written behind
    the last start."""
    b = Batch([(rows, 100), (rows, 200)], 2, 32, behind=4)
    q8, qs = queries(b.rng, b.rows, 4)
    want, mag, top = attend(b, q8, qs, 4, QK)
    pool, _ = on_device(b)
    kv_len = b.kv_len.copy()
    for wrong in (1 << 30, 2147483647, -5, -2147483648):
        kv_len[0] = wrong
        seqs = ops.sequences(pool, dev(b.tables), dev(b.start), dev(kv_len), b.max_rows, b.max_kv)
        out = torch.full((b.rows, 512), 7.5, device="cuda")
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
        got = out.cpu().numpy()
        assert (np.abs(got - want) <= attend_bound(mag, top, b.max_kv))[rows:2 * rows].all()
        assert (got[2 * rows:] == 7.5).all()
    for start in ([0, rows, 1 << 30], [-7, rows, 2 * rows], [-2147483648, 2147483647, 2 * rows], [2 * rows, rows, 0]):
        seqs = ops.sequences(pool, dev(b.tables), dev(np.array(start, np.int32)), dev(b.kv_len), b.max_rows, b.max_kv)
        out = torch.full((b.rows + 8, 512), 7.5, device="cuda")
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
        assert (out.cpu().numpy()[b.rows:] == 7.5).all()


def test_attention_scales(cuda):
    """Query scales of zero and below zero; one key scale that outweighs the rest;
    subnormal and large V scales."""
    b = Batch([(1, 300), (37, 90)], 2, 32, seed=3)
    s = b.rng.integers(0, b.n_pages, 5)
    b.ks[s, 3] *= 40
    for i in range(2):
        t = np.arange(int(b.kv_len[i]))
        at = b.tables[i, t // 32], t % 32
        b.vs[at] *= np.where(t % 7 == 0, F(1e-38), np.where(t % 7 == 1, F(1e30), F(1)))[:, None].astype(F)
    q8, qs = queries(b.rng, b.rows, 4)
    qs[::3] = 0
    qs[1::3] *= -1
    want, mag, top = attend(b, q8, qs, 4, QK)
    pool, seqs = on_device(b)
    out = torch.empty((b.rows, 512), device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
    got = out.cpu().numpy()
    err, bound = np.abs(got - want), attend_bound(mag, top, b.max_kv)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("kind", ["few", "short", "many", "hole", "wide", "listed"])
def test_attention_unsplit(cuda, kind):
    """So many sequences (of the same pages) that their 17000 keys are not split: more
    blocks than are named at a time."""
    kvh, n_sel = 16, 300
    n, rows = {"few": (100, 1), "listed": (100, 1), "short": (49, 17)}.get(kind, (50, 49))
    b = Batch([(rows, 17000 - rows)], kvh, 32, seed=6)
    if kind == "hole":
        b.tables[0, 300:310] = 65535
    if kind == "wide":
        b.vs *= np.exp2(np.floor(b.rng.random(b.vs.shape) * 12) - 6).astype(F)
    q8, qs = queries(b.rng, n * rows, kvh)
    lens = 17000 - 7 * np.arange(n)
    ids = np.sort(np.stack([b.rng.permutation(531)[:n_sel] for _ in range(kvh)]), 1).astype(np.int32).reshape(1, -1)
    pool, _ = on_device(b)
    seqs = ops.sequences(pool, dev(np.repeat(b.tables, n, 0)), dev((rows * np.arange(n + 1)).astype(np.int32)),
                         dev(lens.astype(np.int32)), rows, 17000)
    out = torch.empty((n * rows, kvh * 128), device="cuda")
    if kind == "listed":
        ops.attention_pages(dev(q8), dev(qs), pool, seqs, dev(np.repeat(ids, n, 0)), n_sel, out, qk_scale=QK)
    else:
        ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
    got = out.cpu().numpy()
    assert np.isfinite(got).all()
    for i in (0, n // 2, n - 1):
        b.lens, b.kv_len, b.rows = [(rows, int(lens[i]) - rows)], lens[i:i + 1], rows
        at = slice(i * rows, (i + 1) * rows)
        want, mag, top = attend(b, q8[at], qs[at], kvh, QK, True, ids if kind == "listed" else None, n_sel)
        assert (np.abs(got[at] - want) <= attend_bound(mag, top, 17000)).all(), i


@pytest.mark.parametrize("lens,heads,kv_heads", [([(1, 543)], 16, 8), ([(1, 700), (1, 5), (1, 1300)], 16, 8), ([(33, 500), (1, 90)], 16, 8),
                                                 ([(300, 500), (1, 40)], 16, 2)])
def test_attention_loose_limits(cuda, lens, heads, kv_heads):
    """max_kv far above the lengths, tables as wide: the same results, and a workspace
    that does not grow with it without end."""
    b = Batch(lens, kv_heads, 32, seed=12)
    q8, qs = queries(b.rng, b.rows, heads)
    pool, seqs = on_device(b)
    wide = np.full((len(lens), 8192), 65535, np.uint16)
    wide[:, :b.tables.shape[1]] = b.tables
    loose = ops.sequences(pool, dev(wide), *seqs._keep[1:], b.max_rows, 8192 * 32)
    assert ops.seqs_workspace_bytes(pool, loose, b.rows, heads) <= 65 * (b.rows + 128 * len(lens)) * heads * 520
    want, mag, top = attend(b, q8, qs, heads, QK)
    out = torch.empty((b.rows, heads * 128), device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, loose, out, qk_scale=QK)
    assert (np.abs(out.cpu().numpy() - want) <= attend_bound(mag, top, b.max_kv)).all()


@pytest.mark.parametrize("lens,heads,kv_heads", [([(24, 4000)] * 10, 16, 8), ([(5, 3000), (1, 5000), (48, 700), (0, 9), (17, 0)] * 5, 8, 8),
                                                 ([(4, 2000), (1, 3500), (6, 100)] * 6, 64, 8)])
def test_attention_short_chunks(cuda, lens, heads, kv_heads):
    """Up to 48 columns of every sequence: 16-column tiles alone, some of them split."""
    b = Batch(lens, kv_heads, 32, seed=14)
    assert b.rows * heads * b.max_kv > 12 << 20 and b.max_rows * heads // kv_heads <= 48
    check_attention(b, heads)


@pytest.mark.parametrize("n", [64, 65, 128, 129, 700, 4096])
def test_many_sequences(cuda, n):
    """More sequences than a wave has lanes, some without rows, rows around them all."""
    lens = [((i * 7) % 3, (i * 13) % 40) for i in range(n)]
    if n == 129:
        lens[70] = (2000, 700)  # 128-column tiles too
    b = Batch(lens, 2, 32, seed=n, before=3, behind=2)
    check_attention(b, 4)
    append_case(Batch(lens, 2, 32, seed=n, before=3, behind=2), 4, 64, False, True)
    bounds, scale, _ = bounds_on_host(b)
    q8, qs = queries(b.rng, b.rows, 4)
    pool, seqs = on_device(b)
    ids = torch.full((b.rows, 2), 7, dtype=torch.int32, device="cuda")
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, 1)
    want = np.full((b.rows, 2), 7, np.int32)
    for row, _, pos in b.row_positions():
        want[row] = pos // 32
    assert np.array_equal(ids.cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["few", "many", "listed"])
def test_attention_nan(cuda, kind):
    """A NaN query, key or value scale reaches the results that it enters, whole rows of
    a head, and no other."""
    lens, page = ([(800, 300), (1, 40), (100, 700)] if kind == "many" else [(5, 700), (1, 40), (3, 2)]), 32
    b = Batch(lens, 2, page, seed=4)
    heads = 16 if kind == "many" else 4
    assert (b.rows * heads * b.max_kv > 12 << 20) == (kind == "many")
    q8, qs = queries(b.rng, b.rows, heads)
    n_sel = 4
    ids = np.tile(np.arange(n_sel, dtype=np.int32), (b.rows, 2))
    pool, seqs = on_device(b)
    tq = dev(q8)

    def run(pool, qs):
        out = torch.empty((b.rows, heads * 128), device="cuda")
        if kind == "listed":
            ops.attention_pages(tq, dev(qs), pool, seqs, dev(ids), n_sel, out, qk_scale=QK)
        else:
            ops.attention_varlen_paged(tq, dev(qs), pool, seqs, out, qk_scale=QK)
        return out.cpu().numpy().reshape(b.rows, heads, 128)

    plain = run(pool, qs)
    assert np.isfinite(plain).all()
    _, mag, top = attend(b, q8, qs, heads, QK, True, ids if kind == "listed" else None, n_sel)
    # both runs are within the bound of the same value
    twice = 2 * attend_bound(mag, top, b.max_kv).reshape(plain.shape)
    bad = qs.copy()
    bad[::2, 1] = np.nan
    got, want = run(pool, bad), plain.copy()
    want[::2, 1] = np.nan
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert (np.abs(got - want) <= twice)[~np.isnan(want)].all()
    rows = {r: (s, p) for r, s, p in b.row_positions()}
    for name in ("ks", "vs"):
        t = 33  # of sequence 0, KV head 1: the heads of the upper half
        keep = getattr(b, name).copy()
        getattr(b, name)[b.tables[0, t // page], t % page, 1] = np.nan
        got, want = run(on_device(b)[0], qs), plain.copy()
        sees = [r for r, (s, p) in rows.items() if s == 0 and p >= t]
        want[sees, heads // 2:] = np.nan
        same = np.isnan(got) == np.isnan(want)
        assert same.all(), np.argwhere(~same)[:4].tolist()
        assert (np.abs(got - want) <= twice)[~np.isnan(want)].all()
        getattr(b, name)[:] = keep


def test_attention_strided(cuda):
    """Query and result rows inside wider ones."""
    b = Batch([(5, 60), (1, 700), (50, 0)], 2, 32, seed=4)
    q8, qs = queries(b.rng, b.rows, 4)
    want, mag, top = attend(b, q8, qs, 4, QK)
    pool, seqs = on_device(b)
    wq = torch.zeros((b.rows, 4 * 128 + 48), dtype=torch.int8, device="cuda")
    wq[:, 16:16 + 512] = dev(q8)
    ws = torch.zeros((b.rows, 9), device="cuda")
    ws[:, 2:6] = dev(qs)
    wo = torch.full((b.rows, 512 + 7), 7.5, device="cuda")
    ops.attention_varlen_paged(wq[:, 16:528], ws[:, 2:6], pool, seqs, wo[:, 3:515], qk_scale=QK)
    got = wo.cpu().numpy()
    assert (np.abs(got[:, 3:515] - want) <= attend_bound(mag, top, b.max_kv)).all()
    assert (got[:, :3] == 7.5).all() and (got[:, 515:] == 7.5).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_far_pages(cuda, rows):
    """Pages whose bytes lie behind 2^32 of a long cache."""
    n_pages, page, kvh = 20000, 256, 8
    b = Batch([(rows, 700)], kvh, page, seed=6)
    k = torch.empty((n_pages, page, kvh * 128), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty((n_pages, page, kvh), device="cuda")
    vs = torch.empty_like(ks)
    far = n_pages - b.n_pages
    k[far:], v[far:] = dev(b.k).view(b.n_pages, page, -1), dev(b.v).view(b.n_pages, page, -1)
    ks[far:], vs[far:] = dev(b.ks), dev(b.vs)
    pool = ops.kv_pool(k, v, ks, vs)
    seqs = ops.sequences(pool, dev((b.tables.astype(np.int64) + far).astype(np.uint16)), dev(b.start), dev(b.kv_len),
                         b.max_rows, b.max_kv)
    q8, qs = queries(b.rng, b.rows, 16)
    out = torch.empty((b.rows, 2048), device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
    want, mag, top = attend(b, q8, qs, 16, QK)
    assert (np.abs(out.cpu().numpy() - want) <= attend_bound(mag, top, b.max_kv)).all()
    x = torch.randn((b.rows, 3 * 1024), device="cuda")
    ops.rope_append_paged(None, x[:, :1024], x[:, 1024:2048], pool, seqs)
    r8, rs = quantise(x[:, :1024].cpu().numpy())
    pos = b.kv_len[0] - rows + np.arange(rows)
    p = dev(b.tables[0, pos // page].astype(np.int64) + far)
    assert bits_equal(k[p, dev(pos % page)].cpu().numpy(), r8) and bits_equal(ks[p, dev(pos % page)].cpu().numpy(), rs)


@pytest.mark.parametrize("heads,kv_heads,page,n_sel", [(16, 8, 32, 4), (6, 2, 96, 1), (16, 1, 32, 7), (64, 2, 64, 40), (33, 1, 32, 5)])
def test_attention_pages(cuda, heads, kv_heads, page, n_sel):
    """Listed pages in any order; ids that name none of the row's pages are passed
    over, a page listed twice counts twice; rows with no page at all."""
    b = Batch([(1, 900), (7, 300), (1, 0), (20, 1500), (3, -2)], kv_heads, page, seed=heads, before=1, behind=2)
    ids = b.rng.integers(-2, b.tables.shape[1] + 2, (b.rows, kv_heads * n_sel)).astype(np.int32)
    ids[3] = -1
    ids[5, :] = ids[5, 0]
    ids[6, ::2] = 2147483647
    ids[7, ::2] = -2147483648
    check_attention(b, heads, ids=ids, n_sel=n_sel)


# ---- appending ----------------------------------------------------------------


def append_case(b, heads, rot, interleaved, norm, fused=True, seed=0):
    """Runs the append and its plain form; returns what the device holds."""
    rng, kvh = np.random.default_rng(seed), b.kv_heads
    x = rng.standard_normal((b.rows, (heads + 2 * kvh) * 128 + 1)).astype(F)
    x[0, :128] = 0
    off = 0 if fused else 1  # 1: rows that no 16-byte word fits
    tx = dev(x)[:, off:off + (heads + 2 * kvh) * 128]
    xn = x[:, off:off + (heads + 2 * kvh) * 128]
    if fused:
        tx = tx.contiguous()
    q, k, v = tx[:, :heads * 128], tx[:, heads * 128:(heads + kvh) * 128], tx[:, (heads + kvh) * 128:]
    nw = [(1 + 0.1 * rng.standard_normal(128)).astype(F) for _ in range(2)]
    cos, sin = rope_tables(max(b.max_kv, 1), rot) if rot else (None, None)
    pool, seqs = on_device(b)
    q8 = torch.full((b.rows, heads * 128), 99, dtype=torch.int8, device="cuda")
    qs = torch.full((b.rows, heads), 7.5, device="cuda")
    ops.rope_append_paged(q, k, v, pool, seqs, q8, qs, nwq=dev(nw[0]) if norm else None, nwk=dev(nw[1]) if norm else None,
                          inv_hd=1 / 128, cos=dev(cos) if rot else None, sin=dev(sin) if rot else None, rot_dim=rot,
                          interleaved=interleaved)
    want = dict(q8=np.full((b.rows, heads * 128), 99, np.int8), qs=np.full((b.rows, heads), 7.5, F),
                k=b.k.copy(), ks=b.ks.copy(), v=b.v.copy(), vs=b.vs.copy())
    for row, s, pos in b.row_positions():
        if pos < 0:
            continue
        r = xn[row].reshape(-1, 128)
        for name, h0, h1, w in (("q", 0, heads, nw[0]), ("k", heads, heads + kvh, nw[1]), ("v", heads + kvh, heads + 2 * kvh, None)):
            y = r[h0:h1]
            if name != "v":
                y = seqref.head_norm(y, w) if norm else y
                y = seqref.rotate(y, cos[pos], sin[pos], rot, interleaved) if rot else y
            y8, ys = quantise(y.reshape(1, -1))
            if name == "q":
                want["q8"][row], want["qs"][row] = y8[0], ys[0]
            elif b.tables[s, pos // b.page] < b.n_pages:
                at = b.tables[s, pos // b.page], pos % b.page
                want[name][at], want[name + "s"][at] = y8.reshape(-1, 128), ys[0]
    tk, tv, tks, tvs = pool._keep
    got = dict(q8=q8, qs=qs, k=tk, ks=tks, v=tv, vs=tvs)
    for n, t in got.items():
        g, w = t.cpu().numpy(), want[n]
        assert bits_equal(g.reshape(w.shape), w), (n, describe_diff(g.reshape(w.shape), w))
    return pool, seqs, want


@pytest.mark.parametrize("lens", ["one", "decode", "chunks", "empty_ones", "none_before", "page_edges"])
@pytest.mark.parametrize("heads,kv_heads,page", [(16, 8, 32), (5, 3, 96)])
def test_append(cuda, lens, heads, kv_heads, page):
    append_case(Batch(LENS[lens], kv_heads, page, seed=2, before=2, behind=3), heads, 128, False, True)


@pytest.mark.parametrize("rot", [0, 2, 6, 32, 64, 96, 100, 126, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_append_rotations(cuda, rot, interleaved, fused):
    append_case(Batch([(7, 50), (1, 31), (1, 4000)], 2, 32, seed=rot), 4, rot, interleaved, rot % 4 == 0, fused, seed=rot)


def test_append_norm_factor(cuda):
    """The norm's factor is that of heads of 128 if none is given."""
    b = Batch([(3, 30)], 2, 32)
    x, w = torch.randn((3, 512), device="cuda"), torch.rand(128, device="cuda")
    res = []
    for kw in ({}, {"inv_hd": 1 / 128}):
        pool, seqs = on_device(b)
        q8, qs = torch.empty((3, 512), dtype=torch.int8, device="cuda"), torch.empty((3, 4), device="cuda")
        ops.rope_append_paged(x, x[:, :256], x[:, 256:], pool, seqs, q8, qs, nwq=w, nwk=w, **kw)
        res.append((q8, qs, *(t.nan_to_num() for t in pool._keep)))
    assert all(torch.equal(s, t) for s, t in zip(*res))


def test_append_bad_pages(cuda):
    b = Batch([(40, 20), (1, 64)], 2, 32)
    b.tables[0, 1] = b.n_pages
    append_case(b, 4, 128, False, True)


def test_append_keys_alone(cuda):
    b = Batch([(4, 30), (1, 5)], 2, 32)
    pool, seqs = on_device(b)
    x = torch.randn((b.rows, 256), device="cuda")
    ops.rope_append_paged(None, x, x, pool, seqs)
    r8, rs = quantise(x.cpu().numpy())
    for row, s, pos in b.row_positions():
        at = int(b.tables[s, pos // 32]), pos % 32
        for i in (0, 1):
            assert bits_equal(pool._keep[i][at].cpu().numpy(), r8[row]) and bits_equal(pool._keep[2 + i][at].cpu().numpy(), rs[row])


def test_append_equals_norm_rope_quant_heads(cuda):
    """Bit for bit what the one-sequence operator gives for the same rows."""
    b = Batch([(60, 77)], 8, 32)
    rng = np.random.default_rng(0)
    x = dev((5 * rng.standard_normal((60, 32 * 128))).astype(F))
    w = dev((1 + 0.1 * rng.standard_normal(128)).astype(F))
    cos, sin = (dev(t) for t in rope_tables(b.max_kv))
    pool, seqs = on_device(b)
    q8, qs = torch.empty((60, 2048), dtype=torch.int8, device="cuda"), torch.empty((60, 16), device="cuda")
    q, k, v = x.split([2048, 1024, 1024], 1)
    ops.rope_append_paged(q, k, v, pool, seqs, q8, qs, nwq=w, nwk=w, inv_hd=1 / 128, cos=cos, sin=sin)
    for heads, rows, got, gs in ((16, q, q8, qs), (8, k, None, None)):
        r8, rs = torch.empty((60, heads * 128), dtype=torch.int8, device="cuda"), torch.empty((60, heads), device="cuda")
        ops.norm_rope_quant_heads(rows, w, cos[77:], sin[77:], r8, rs, heads, 1 / 128)
        if got is None:
            t = np.arange(77, 137)
            p = dev(b.tables[0, t // 32].astype(np.int64))
            got, gs = pool._keep[0][p, dev(t % 32)], pool._keep[2][p, dev(t % 32)]
        assert torch.equal(got, r8) and torch.equal(gs, rs)


# ---- page bounds and selection ---------------------------------------------------


def bounds_on_host(b):
    """Bounds of every page of the batch's sequences."""
    bounds = np.full((b.n_pages * b.kv_heads, 256), 5, np.int8)
    scale = np.full((b.n_pages, b.kv_heads), 7.5, F)
    touched = np.zeros(b.n_pages, bool)
    for s, (n, _) in enumerate(b.lens):
        kv = int(b.kv_len[s])
        for i in range(-(-max(kv, 0) // b.page)):
            p, tokens = int(b.tables[s, i]), min(b.page, kv - i * b.page)
            if p >= b.n_pages:
                continue
            touched[p] = n > 0 and (i + 1) * b.page > kv - n
            for h in range(b.kv_heads):
                bounds[p * b.kv_heads + h], scale[p, h] = seqref.bounds_of(b.k[p, :tokens, h], b.ks[p, :tokens, h])
    return bounds, scale, touched


@pytest.mark.parametrize("lens", ["one", "decode", "chunks", "empty_ones", "none_before", "page_edges"])
@pytest.mark.parametrize("kv_heads,page", [(8, 32), (3, 96), (2, 256)])
def test_page_bounds(cuda, lens, kv_heads, page):
    b = Batch(LENS[lens], kv_heads, page, seed=9)
    want, wscale, touched = bounds_on_host(b)
    pool, seqs = on_device(b)
    bounds = torch.full(want.shape, 5, dtype=torch.int8, device="cuda")
    scale = torch.full(wscale.shape, 7.5, device="cuda")
    ops.page_bounds(pool, seqs, bounds, scale, b.rows)
    got, gs = bounds.cpu().numpy().reshape(b.n_pages, -1), scale.cpu().numpy()
    w = want.reshape(b.n_pages, -1)
    assert bits_equal(got[touched], w[touched]) and bits_equal(gs[touched], wscale[touched])
    assert (got[~touched] == 5).all() and (gs[~touched] == 7.5).all()


def test_page_bounds_bound_the_scores(cuda):
    """q . k * qs * ks of every key is at most its page's score, within the f32
    roundings of the scale (2^-23) and of the score (2^-23)."""
    b = Batch([(64, 0)], 2, 32, seed=11)
    pool, seqs = on_device(b)
    bounds, scale = torch.zeros((b.n_pages * 2, 256), dtype=torch.int8, device="cuda"), torch.zeros((b.n_pages, 2), device="cuda")
    ops.page_bounds(pool, seqs, bounds, scale, b.rows)
    bh, sh = bounds.cpu().numpy().astype(np.float64), scale.cpu().numpy().astype(np.float64)
    q = b.rng.integers(-127, 128, (50, 128)).astype(np.float64)
    for i in range(2):
        p = int(b.tables[0, i])
        for h in range(2):
            k = b.k[p, :, h].astype(np.float64) * b.ks[p, :, h][:, None].astype(np.float64)
            lo, hi = bh[p * 2 + h, :128], bh[p * 2 + h, 128:]
            top = (np.where(q > 0, hi, lo) * q).sum(1) * sh[p, h]
            room = np.abs(q).sum(1) * 127 * sh[p, h] * 2.0 ** -22
            assert ((q @ k.T).max(1) <= top + room).all()


@pytest.mark.parametrize("heads,kv_heads,page,n_sel", [(16, 8, 32, 4), (6, 2, 96, 1), (16, 1, 32, 7), (32, 2, 64, 33), (20, 4, 32, 20), (2, 2, 32, 300)])
def test_select_pages(cuda, heads, kv_heads, page, n_sel):
    b = Batch([(1, 2900), (7, 300), (1, 0), (20, 1500), (3, -2), (0, 40), (1, 5000)], kv_heads, page, seed=heads, before=1, behind=2, smooth=True)
    b.tables[0, 5] = 65535
    bounds, scale, _ = bounds_on_host(b)
    q8, qs = queries(b.rng, b.rows, heads)
    pool, seqs = on_device(b)
    ids = torch.full((b.rows, kv_heads * n_sel), -9, dtype=torch.int32, device="cuda")
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, n_sel)
    want = seqref.select(b, q8, qs, heads, bounds, scale, n_sel)
    assert np.array_equal(ids.cpu().numpy(), want), np.argwhere(ids.cpu().numpy() != want)[:5]


@pytest.mark.parametrize("n_sel", [1, 2, 17, 255, 256, 257, 300])
def test_select_ties(cuda, n_sel):
    """Few distinct scores: equal ones go to the lowest pages, over many waves."""
    b = Batch([(1, 32 * 300 + 3), (2, 32 * 290)], 2, 32, seed=n_sel)
    bounds = np.repeat(b.rng.integers(-2, 3, (b.n_pages * 2, 1)), 256, 1).astype(np.int8)
    scale = np.full((b.n_pages, 2), 0.5, F)
    q8 = np.ones((b.rows, 4 * 128), np.int8)
    qs = np.full((b.rows, 4), 0.25, F)
    qs[1] = 0  # all scores are zeros of either sign
    pool, seqs = on_device(b)
    ids = torch.empty((b.rows, 2 * n_sel), dtype=torch.int32, device="cuda")
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, n_sel)
    want = seqref.select(b, q8, qs, 4, bounds, scale, n_sel)
    assert np.array_equal(ids.cpu().numpy(), want)


@pytest.mark.parametrize("pages", [4095, 4096, 4097, 6000])
def test_select_many_pages(cuda, pages):
    """Both sides of what the keys' registers hold; a table that names its few pages
    over and over, so most scores tie."""
    b = Batch([(1, 32 * 40), (2, 32 * 20)], 2, 32, seed=pages)
    b.tables = b.rng.integers(0, b.n_pages, (2, pages)).astype(np.uint16)
    b.kv_len = np.array([32 * pages - 5, 32 * (pages - 1) + 1], np.int32)
    b.lens = [(1, int(b.kv_len[0]) - 1), (2, int(b.kv_len[1]) - 2)]
    b.max_kv = int(b.kv_len.max())
    bounds = b.rng.integers(-127, 128, (b.n_pages * 2, 256)).astype(np.int8)
    scale = b.rng.uniform(0.1, 1, (b.n_pages, 2)).astype(F)
    q8, qs = queries(b.rng, b.rows, 6)
    pool, seqs = on_device(b)
    for n_sel in (5, 700):
        ids = torch.empty((b.rows, 2 * n_sel), dtype=torch.int32, device="cuda")
        ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, n_sel)
        assert np.array_equal(ids.cpu().numpy(), seqref.select(b, q8, qs, 6, bounds, scale, n_sel))


def test_select_extremes(cuda):
    """Scores of the int8 limits (-128 included), NaN scales first of all, -inf last."""
    b = Batch([(1, 32 * 40)], 1, 32, seed=1)
    bounds = b.rng.integers(-128, 128, (b.n_pages, 256)).astype(np.int8)
    scale = b.rng.uniform(0.1, 1, (b.n_pages, 1)).astype(F)
    t = b.tables[0]
    scale[t[7]] = np.nan
    scale[t[9]] = -np.inf
    bounds[t[9], 128:] = 127
    q8 = np.full((1, 256), -128, np.int8)
    q8[0, 128:] = 127
    qs = np.ones((1, 2), F)
    pool, seqs = on_device(b)
    ids = torch.empty((1, 40), dtype=torch.int32, device="cuda")
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, 2)
    assert ids[0, :2].tolist() == [7, 40]
    scale[t[7]] = 0.5
    scale[t[9]] = 0.0
    ids.fill_(-9)
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(bounds), dev(scale), ids, 40)
    assert np.array_equal(ids.cpu().numpy(), seqref.select(b, q8, qs, 2, bounds, scale, 40))


# ---- together --------------------------------------------------------------------


def test_steps_together(cuda):
    """Prompt chunks, then decoding steps: each step's rows appended, their pages'
    bounds refreshed, dense attention and attention over chosen pages, all against
    the plain forms on the cache as it then is."""
    heads, kvh, page, n_sel = 8, 2, 32, 3
    b = Batch([(40, 0), (75, 0), (1, 200)], kvh, page, seed=20)
    b.max_kv += 4
    b.tables = np.concatenate((b.tables, np.full((3, 1), 65535, np.uint16)), 1)
    cos, sin = rope_tables(b.max_kv, scaling="yarn", factor=4.0, original=64)
    rng = np.random.default_rng(0)
    pool, _ = on_device(b, max_kv=1)
    tk, tv, tks, tvs = pool._keep
    bounds = torch.zeros((b.n_pages * kvh, 256), dtype=torch.int8, device="cuda")
    scale = torch.zeros((b.n_pages, kvh), device="cuda")
    # the third sequence's old pages
    old = ops.sequences(pool, dev(b.tables), dev(np.array([0, 0, 0, 200], np.int32)), dev(np.array([0, 0, 200], np.int32)), 200, 200)
    ops.page_bounds(pool, old, bounds, scale, 200)
    free = [p for p in range(b.n_pages) if p not in b.tables]
    for step in range(3):
        rows = int(b.start[-1])
        x = rng.standard_normal((rows, (heads + 2 * kvh) * 128)).astype(F)
        tx = dev(x)
        seqs = ops.sequences(pool, dev(b.tables), dev(b.start), dev(b.kv_len), max(r for r, _ in b.lens), b.max_kv)
        q8, qs = torch.empty((rows, heads * 128), dtype=torch.int8, device="cuda"), torch.empty((rows, heads), device="cuda")
        ops.rope_append_paged(tx[:, :1024], tx[:, 1024:1280], tx[:, 1280:], pool, seqs, q8, qs, cos=dev(cos), sin=dev(sin))
        ops.page_bounds(pool, seqs, bounds, scale, rows)
        out, sparse = torch.empty((rows, heads * 128), device="cuda"), torch.empty((rows, heads * 128), device="cuda")
        ids = torch.empty((rows, kvh * n_sel), dtype=torch.int32, device="cuda")
        ws = torch.empty(max(16, ops.seqs_workspace_bytes(pool, seqs, rows, heads, n_sel)), dtype=torch.uint8, device="cuda")
        ops.attention_varlen_paged(q8, qs, pool, seqs, out, qk_scale=QK, workspace=ws)
        ops.select_pages(q8, qs, pool, seqs, bounds, scale, ids, n_sel, workspace=ws)
        ops.attention_pages(q8, qs, pool, seqs, ids, n_sel, sparse, qk_scale=QK, workspace=ws)
        b.k, b.v = (t.cpu().numpy().reshape(b.n_pages, page, kvh, 128) for t in (tk, tv))
        b.ks, b.vs = tks.cpu().numpy(), tvs.cpu().numpy()
        hb, hs, _ = bounds_on_host(b)
        hq, hqs = q8.cpu().numpy(), qs.cpu().numpy()
        for row, s, pos in b.row_positions():  # the rows that were appended are the ones in the cache
            y = x[row, 1024:1280].reshape(kvh, 128)
            r8, rs = quantise(seqref.rotate(y, cos[pos], sin[pos], 128, False).reshape(1, -1))
            at = b.tables[s, pos // page], pos % page
            assert bits_equal(b.k[at].reshape(-1), r8[0]) and bits_equal(b.ks[at], rs[0])
        want, mag, top = attend(b, hq, hqs, heads, QK)
        assert (np.abs(out.cpu().numpy() - want) <= attend_bound(mag, top, b.max_kv)).all()
        wids = seqref.select(b, hq, hqs, heads, hb, hs, n_sel)
        assert np.array_equal(ids.cpu().numpy(), wids)
        want, mag, top = attend(b, hq, hqs, heads, QK, ids=wids, n_sel=n_sel)
        assert (np.abs(sparse.cpu().numpy() - want) <= attend_bound(mag, top, b.max_kv)).all()
        # one decoding token each
        b.lens = [(1, int(n)) for n in b.kv_len]
        b.start = np.arange(4, dtype=np.int32)
        b.kv_len = b.kv_len + 1
        b.rows = 3
        for s in range(3):
            if b.tables[s, (int(b.kv_len[s]) - 1) // page] == 65535:
                b.tables[s, (int(b.kv_len[s]) - 1) // page] = free.pop()


@pytest.mark.parametrize("rows,context", [(1, 500), (33, 500), (300, 1600)])
def test_captured_and_replayed(cuda, rows, context):
    """A step captured once and replayed on other lengths, tables and rows, with
    eager calls of the same operators between the replays; two graphs that share
    a workspace, replayed in turn."""
    heads, kvh, page, n_sel, n = 8, 4, 32, 4, 3  # (300 rows: the 128-column tiles too)
    b = Batch([(rows, context)] * n, kvh, page, seed=30, smooth=True)
    pool, _ = on_device(b)
    tk, tv, tks, tvs = pool._keep
    total, max_kv = n * rows, b.max_kv
    tables, start, kv_len = dev(b.tables), dev(b.start), dev(b.kv_len)
    seqs = ops.sequences(pool, tables, start, kv_len, rows, max_kv)
    hb, hs, _ = bounds_on_host(b)
    bounds, scale = dev(hb), dev(hs)
    q8, qs = (dev(t) for t in queries(b.rng, total, heads))
    ws = torch.empty(max(16, ops.seqs_workspace_bytes(pool, seqs, total, heads, n_sel)), dtype=torch.uint8, device="cuda")

    def step(o, ids, sp, w):
        ops.attention_varlen_paged(q8, qs, pool, seqs, o, qk_scale=QK, workspace=w)
        ops.select_pages(q8, qs, pool, seqs, bounds, scale, ids, n_sel, workspace=w)
        ops.attention_pages(q8, qs, pool, seqs, ids, n_sel, sp, qk_scale=QK, workspace=w)

    new = lambda: (torch.empty((total, heads * 128), device="cuda"),  # noqa: E731
                   torch.empty((total, kvh * n_sel), dtype=torch.int32, device="cuda"), torch.empty((total, heads * 128), device="cuda"))
    sets, graphs = [new(), new()], []
    side = torch.cuda.Stream()
    for s in sets:
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            step(*s, ws)
        graphs.append(g)
    for lens in ([(rows, 400)] * n, [(rows, 0), (rows, 90), (rows, 500)], [(0, 40), (rows, 33), (1, 31)], [(rows, context)] * n):
        kv_len.copy_(torch.tensor([r + c for r, c in lens], dtype=torch.int32))
        start.copy_(torch.tensor(np.cumsum([0] + [r for r, _ in lens]).astype(np.int32)))
        eager = new()
        for t in (*sets[0], *sets[1], *eager):
            t.zero_()
        graphs[0].replay()
        step(*eager, None)
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for s in sets:
            for got, want in zip(s, eager):
                assert torch.equal(got, want), lens


@pytest.mark.parametrize("rows", [1, 70])
def test_append_captured_and_replayed(cuda, rows):
    """Rows appended, and their pages bounded, by a graph on other lengths, rows and
    inputs, step after step, beside eager calls on a pool of the same contents."""
    heads, kvh, page, n = 4, 2, 32, 3
    b = Batch([(rows, 400)] * n, kvh, page, seed=31)
    b.ks[:], b.vs[:] = np.nan_to_num(b.ks), np.nan_to_num(b.vs)
    pools = [on_device(b)[0] for _ in range(2)]
    total = n * rows
    start, kv_len = dev(b.start), dev(b.kv_len)
    seqs = ops.sequences(pools[0], dev(b.tables), start, kv_len, rows, b.max_kv)
    cos, sin = (dev(t) for t in rope_tables(b.max_kv))
    x = [torch.randn((total, h * 128), device="cuda") for h in (heads, kvh, kvh)]
    res = [(torch.zeros((total, heads * 128), dtype=torch.int8, device="cuda"), torch.zeros((total, heads), device="cuda"),
            torch.zeros((b.n_pages * kvh, 256), dtype=torch.int8, device="cuda"), torch.zeros((b.n_pages, kvh), device="cuda")) for _ in pools]

    def step(i):
        ops.rope_append_paged(*x, pools[i], seqs, *res[i][:2], cos=cos, sin=sin)
        ops.page_bounds(pools[i], seqs, *res[i][2:], total)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(0)
    for lens in ([(rows, 300)] * n, [(rows, 0), (0, 31), (rows, 90)], [(1, 31), (rows, 331), (1, 0)], [(rows, 400)] * n):
        kv_len.copy_(torch.tensor([r + c for r, c in lens], dtype=torch.int32))
        start.copy_(torch.tensor(np.cumsum([0] + [r for r, _ in lens]).astype(np.int32)))
        for t in x:
            t.normal_()
        g.replay()
        step(1)
        torch.cuda.synchronize()
        for got, want in zip((*pools[0]._keep, *res[0]), (*pools[1]._keep, *res[1])):
            assert torch.equal(got, want), lens


def test_selection_on_two_streams(cuda):
    """The selection and the attention over its pages on two streams at once, each with
    its own workspace, which all their calls share in turn."""
    heads, kvh, n_sel = 8, 4, 5
    b = Batch([(1, 3000), (20, 1000)], kvh, 32, seed=41, smooth=True)
    pool, seqs = on_device(b)
    hb, hs, _ = bounds_on_host(b)
    bounds, scale = dev(hb), dev(hs)
    q8, qs = (dev(t) for t in queries(b.rng, b.rows, heads))
    n = ops.seqs_workspace_bytes(pool, seqs, b.rows, heads, n_sel)
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [[(torch.zeros((b.rows, kvh * n_sel), dtype=torch.int32, device="cuda"), torch.zeros((b.rows, heads * 128), device="cuda"))
             for _ in range(4)] for _ in range(3)]
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    for i in range(4):
        for st, w, o in zip([*streams, None], ws, sets):
            ops.select_pages(q8, qs, pool, seqs, bounds, scale, o[i][0], n_sel, workspace=w, stream=st)
            ops.attention_pages(q8, qs, pool, seqs, o[i][0], n_sel, o[i][1], qk_scale=QK, workspace=w, stream=st)
    torch.cuda.synchronize()
    want = seqref.select(b, q8.cpu().numpy(), qs.cpu().numpy(), heads, hb, hs, n_sel)
    assert np.array_equal(sets[2][0][0].cpu().numpy(), want)
    for o in sets:
        for ids, out in o:
            assert torch.equal(ids, sets[2][0][0]) and torch.equal(out, sets[2][0][1])


@pytest.mark.parametrize("n", [3, 100, 700])
def test_bounds_and_selection_of_unequal_sequences(cuda, n):
    """One long chunk among sequences of a row or none: parts of the sequences named one
    by one, and, of many sequences, not."""
    kvh, heads, n_sel = 2, 8, 3
    lens = [(int((i % 5) > 0), (i * 37) % 150) for i in range(n)]
    lens[n // 2] = (300, 200)
    b = Batch(lens, kvh, 32, seed=n, before=1, behind=2, smooth=True)
    pool, seqs = on_device(b)
    want, wscale, touched = bounds_on_host(b)
    bounds = torch.full((b.n_pages * kvh, 256), 99, dtype=torch.int8, device="cuda")
    scale = torch.full(wscale.shape, 7.5, device="cuda")
    ops.page_bounds(pool, seqs, bounds, scale, b.rows)
    got = bounds.cpu().numpy().reshape(b.n_pages, -1)
    assert bits_equal(got[touched], want.reshape(b.n_pages, -1)[touched]) and (got[~touched] == 99).all()
    assert bits_equal(scale.cpu().numpy()[touched], wscale[touched])
    hb = b.rng.integers(-127, 128, (b.n_pages * kvh, 256)).astype(np.int8)
    hs = b.rng.uniform(0.1, 1, (b.n_pages, kvh)).astype(F)
    q8, qs = queries(b.rng, b.rows, heads)
    ids = torch.full((b.rows, kvh * n_sel), 77, dtype=torch.int32, device="cuda")
    ops.select_pages(dev(q8), dev(qs), pool, seqs, dev(hb), dev(hs), ids, n_sel)
    mine = np.zeros(b.rows, bool)
    mine[[r for r, _, _ in b.row_positions()]] = True
    got = ids.cpu().numpy()
    assert np.array_equal(got[mine], seqref.select(b, q8, qs, heads, hb, hs, n_sel)[mine]) and (got[~mine] == 77).all()


def test_page_bounds_rows_given_or_not(cuda):
    """Row starts that do not begin at 0, with and without the call's row count."""
    b = Batch([(1, 40), (33, 31)], 2, 32, before=50)
    pool, seqs = on_device(b)
    want, wscale, touched = bounds_on_host(b)
    for rows in (None, b.rows):
        bounds = torch.full((b.n_pages * 2, 256), 99, dtype=torch.int8, device="cuda")
        scale = torch.full(wscale.shape, 7.5, device="cuda")
        ops.page_bounds(pool, seqs, bounds, scale, rows)
        assert bits_equal(bounds.cpu().numpy().reshape(b.n_pages, -1)[touched], want.reshape(b.n_pages, -1)[touched])
        assert bits_equal(scale.cpu().numpy()[touched], wscale[touched])


def test_two_streams(cuda):
    """Calls of one pool on two streams at once, each with its own workspace."""
    b = Batch([(1, 3000), (40, 100)], 2, 32, seed=40)
    pool, seqs = on_device(b)
    q8, qs = (dev(t) for t in queries(b.rng, b.rows, 4))
    want = torch.empty((b.rows, 512), device="cuda")
    ops.attention_varlen_paged(q8, qs, pool, seqs, want, qk_scale=QK)
    n = max(16, ops.seqs_workspace_bytes(pool, seqs, b.rows, 4))
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in streams]
    outs = [[torch.zeros_like(want) for _ in range(5)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(5):
        for st, w, o in zip(streams, ws, outs):
            ops.attention_varlen_paged(q8, qs, pool, seqs, o[i], qk_scale=QK, workspace=w, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for o in outs for t in o)


def test_no_rows(cuda):
    b = Batch([(0, 40), (0, 0)], 2, 32)
    pool, seqs = on_device(b)
    e = lambda *s, dt=torch.float32: torch.empty(s, dtype=dt, device="cuda")  # noqa: E731
    ops.rope_append_paged(e(0, 512), e(0, 256), e(0, 256), pool, seqs, e(0, 512, dt=torch.int8), e(0, 4))
    ops.page_bounds(pool, seqs, e(b.n_pages * 2, 256, dt=torch.int8), e(b.n_pages, 2), 0)
    ops.attention_varlen_paged(e(0, 512, dt=torch.int8), e(0, 4), pool, seqs, e(0, 512))
    ops.select_pages(e(0, 512, dt=torch.int8), e(0, 4), pool, seqs, e(b.n_pages * 2, 256, dt=torch.int8), e(b.n_pages, 2),
                     e(0, 8, dt=torch.int32), 4)
    none = ops.sequences(pool, e(0, 4, dt=torch.int16), torch.zeros(1, dtype=torch.int32, device="cuda"), e(0, dt=torch.int32), 0, 0)
    out = torch.full((3, 512), 7.5, device="cuda")
    ops.attention_varlen_paged(e(3, 512, dt=torch.int8), e(3, 4), pool, none, out)
    assert (out == 7.5).all()


def test_refused_on_the_device(cuda):
    b = Batch([(1, 40)], 2, 32)
    pool, seqs = on_device(b)
    q8, qs = (dev(t) for t in queries(b.rng, 1, 4))
    out = torch.empty((1, 512), device="cuda")
    with pytest.raises(ValueError):
        ops.attention_varlen_paged(q8.cpu(), qs, pool, seqs, out)
    with pytest.raises(ValueError):
        ops.attention_varlen_paged(q8, qs, pool, seqs, out.t())
    with pytest.raises(ops.Q3Error):
        ops.attention_varlen_paged(q8, qs, pool, seqs, out[:, :511])
    with pytest.raises(ops.Q3Error):
        ops.attention_varlen_paged(q8, qs, pool, seqs)
    with pytest.raises(ValueError):
        ops.kv_pool(*(t[:, :, ::2] for t in pool._keep))
    with pytest.raises(TypeError):
        ops.sequences(pool, seqs._keep[0].int(), *seqs._keep[1:], 1, 41)
    wide = torch.empty((1, 520), device="cuda")
    with pytest.raises(ValueError):
        ops.attention_varlen_paged(wide.to(torch.int8), wide, pool, seqs, wide)
    with pytest.raises(ValueError):
        ops.rope_append_paged(wide, out[:, :256], out[:, :256], pool, seqs, q8, qs)
    fewer = ops.kv_pool(*(t[:-1] for t in pool._keep))  # not all pages that the tables may name
    with pytest.raises(ValueError):
        ops.attention_varlen_paged(q8, qs, fewer, seqs, out)
    with pytest.raises(ValueError):
        ops.rope_append_paged(None, out[:, :256], out[:, :256], fewer, seqs)
    with pytest.raises(ops.Q3Error):
        ops.attention_varlen_paged(q8, qs, pool, ops.sequences(pool, *seqs._keep, -1, 41), out)
    with pytest.raises(ops.Q3Error):
        ops.attention_varlen_paged(q8, qs, pool, ops.sequences(pool, *seqs._keep, 1, 65), out)
    long = Batch([(1, 3000)], 2, 32)
    pool, seqs = on_device(long)
    with pytest.raises(ValueError):  # whose workspace?
        ops.attention_varlen_paged(q8, qs, pool, seqs, out, stream=torch.cuda.Stream())
    for ws in (torch.empty(64, dtype=torch.uint8, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")[4:]):
        with pytest.raises(ops.Q3Error):
            ops.attention_varlen_paged(q8, qs, pool, seqs, out, workspace=ws)
    with pytest.raises(ValueError):
        ops.attention_varlen_paged(q8, qs, pool, seqs, out, workspace=torch.empty(1 << 20, dtype=torch.uint8))
