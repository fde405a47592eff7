"""What the batch operators refuse, and the rotary tables, without a GPU: every
call here must come back before anything is launched.  The data pointers are host
addresses that nothing reads."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from q3ops import _lib
from q3ops.rope import rope_tables
from test_abi_validation import _ADDR, DT_F32, DT_I32, DT_I8, V

OK, ARG, DTYPE, VIEW, UNSUPPORTED, RANGE = 0, -1, -2, -3, -4, -7
F0 = C.c_float(1.0)
H, KV, ROWS = 4, 2, 6


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def pool(**kw):
    p = _lib.PagedKV(_ADDR, _ADDR, _ADDR, _ADDR, None, 32, 32 * 256, 256, 32 * 8, 8)
    for k, v in kw.items():
        setattr(p, k, v)
    return C.byref(p)


def seqs(**kw):
    s = _lib.Seqs(_ADDR, _ADDR, _ADDR, 3, 4, 16, 2, 100)
    for k, v in kw.items():
        setattr(s, k, v)
    return C.byref(s)


BAD_POOL = [(dict(k=None), ARG), (dict(vs=None), ARG), (dict(page_tokens=0), UNSUPPORTED), (dict(page_tokens=48), UNSUPPORTED),
            (dict(page_bytes=32 * 256 - 16), VIEW), (dict(row_bytes=264), VIEW), (dict(row_bytes=128), VIEW),
            (dict(scale_row_bytes=4), VIEW), (dict(scale_row_bytes=10, scale_page_bytes=320), VIEW),
            (dict(scale_page_bytes=32 * 8 - 4), VIEW), (dict(k=_ADDR + 8), VIEW), (dict(ks=_ADDR + 2), VIEW),
            (dict(page_tokens=1 << 31, page_bytes=0xFFFFFFFF), VIEW)]
BAD_SEQS = [(dict(row_start=None), ARG), (dict(kv_len=None), ARG), (dict(tables=None), ARG), (dict(tables=_ADDR + 1), VIEW),
            (dict(row_start=_ADDR + 2), VIEW), (dict(n_seq=65536), RANGE), (dict(n_seq=4097), RANGE), (dict(max_kv=129), RANGE), (dict(ld_table=3), RANGE),
            (dict(max_rows=ROWS + 1), RANGE), (dict(max_kv=(1 << 30) + 1, ld_table=1 << 30), RANGE)]
PLACES = [(pool(**kw), seqs(), rc) for kw, rc in BAD_POOL] + [(pool(), seqs(**kw), rc) for kw, rc in BAD_SEQS] + \
         [(None, seqs(), ARG), (pool(), None, ARG)]


def append(lib, q=V(ROWS, H * 128, DT_F32), k=V(ROWS, KV * 128, DT_F32), v=V(ROWS, KV * 128, DT_F32), nwq=V(128, 1, DT_F32),
           nwk=V(128, 1, DT_F32), cos=V(100, 64, DT_F32), sin=V(100, 64, DT_F32), rot=128, q8=V(ROWS, H * 128, DT_I8),
           qs=V(ROWS, H, DT_F32), kv=pool(), s=seqs(), heads=H, kvh=KV):
    return lib.q3_rope_append_paged(q, k, v, nwq, nwk, F0, cos, sin, rot, 0, q8, qs, kv, s, heads, kvh, None)


def attend(lib, q8=V(ROWS, H * 128, DT_I8), qs=V(ROWS, H, DT_F32), kv=pool(), s=seqs(), out=V(ROWS, H * 128, DT_F32), o8=None,
           os=None, heads=H, kvh=KV, hd=128, ws=None, n=0):
    return lib.q3_attention_varlen_paged(q8, qs, kv, s, out, o8, os, heads, kvh, hd, 1, F0, ws, n, None)


def pages(lib, q8=V(ROWS, H * 128, DT_I8), qs=V(ROWS, H, DT_F32), kv=pool(), s=seqs(), ids=V(ROWS, KV * 3, DT_I32), n_sel=3,
          out=V(ROWS, H * 128, DT_F32), heads=H, kvh=KV, hd=128, ws=None, n=0):
    return lib.q3_attention_pages(q8, qs, kv, s, ids, n_sel, out, None, None, heads, kvh, hd, F0, ws, n, None)


def select(lib, q8=V(ROWS, H * 128, DT_I8), qs=V(ROWS, H, DT_F32), kv=pool(), s=seqs(), bounds=V(32, 256, DT_I8),
           bscale=V(16, 2, DT_F32), ids=V(ROWS, KV * 3, DT_I32), n_sel=3, heads=H, kvh=KV, ws=_ADDR, n=1 << 20):
    return lib.q3_select_pages(q8, qs, kv, s, bounds, bscale, ids, n_sel, heads, kvh, ws, n, None)


def bounds(lib, kv=pool(), s=seqs(), rows=ROWS, kvh=KV, b=V(32, 256, DT_I8), bs=V(16, 2, DT_F32)):
    return lib.q3_page_bounds(kv, s, rows, kvh, b, bs, None)


@pytest.mark.parametrize("call", [append, attend, pages, select, bounds])
def test_pool_and_sequences_refused(lib, call):
    for kv, s, rc in PLACES:
        assert call(lib, kv=kv, s=s) == rc, (kv, s, rc)


def test_append_refused(lib):
    f = V
    for kw, rc in [(dict(k=None), ARG), (dict(v=V(ROWS, KV * 128, DT_I8)), DTYPE), (dict(v=V(ROWS - 1, KV * 128, DT_F32)), VIEW),
                   (dict(k=V(ROWS, KV * 128 - 1, DT_F32)), VIEW), (dict(q=None), ARG), (dict(q8=None), ARG), (dict(qs=None), ARG),
                   (dict(heads=0), ARG), (dict(heads=-1), ARG), (dict(kvh=0), ARG), (dict(q=None, q8=None, qs=None, heads=0), ARG),
                   (dict(q=V(ROWS, H * 128 - 128, DT_F32)), VIEW), (dict(q8=V(ROWS, H * 128 - 1, DT_I8)), VIEW),
                   (dict(q8=V(ROWS, H * 128, DT_I8, row_bytes=H * 128 + 2)), VIEW), (dict(qs=V(ROWS, H - 1, DT_F32)), VIEW),
                   (dict(nwq=V(64, 1, DT_F32)), VIEW), (dict(nwk=V(128, 1, DT_I8)), DTYPE), (dict(cos=None), ARG),
                   (dict(cos=None, sin=None), ARG), (dict(rot=0), ARG), (dict(rot=130), UNSUPPORTED), (dict(rot=63), UNSUPPORTED),
                   (dict(cos=V(99, 64, DT_F32), sin=V(99, 64, DT_F32)), RANGE), (dict(sin=V(100, 65, DT_F32)), VIEW),
                   (dict(cos=V(100, 63, DT_F32), sin=V(100, 63, DT_F32)), VIEW), (dict(kvh=513), ARG)]:
        assert append(lib, **kw) == rc, kw


@pytest.mark.parametrize("call", [attend, pages, select])
def test_queries_refused(lib, call):
    for kw, rc in [(dict(q8=None), ARG), (dict(q8=V(ROWS, H * 128, DT_F32)), DTYPE), (dict(q8=V(ROWS, H * 128 - 16, DT_I8)), VIEW),
                   (dict(q8=V(ROWS, H * 128, DT_I8, row_bytes=H * 128 + 8)), VIEW), (dict(qs=None), ARG),
                   (dict(qs=V(ROWS, H - 1, DT_F32)), VIEW), (dict(qs=V(ROWS - 1, H, DT_F32)), VIEW), (dict(heads=3), ARG),
                   (dict(heads=0), ARG), (dict(kvh=0), ARG), (dict(kvh=-2), ARG)]:
        assert call(lib, **kw) == rc, kw


def test_results_refused(lib):
    for kw, rc in [(dict(out=None), ARG), (dict(o8=V(ROWS, H * 128, DT_I8), os=V(ROWS, H, DT_F32)), ARG),
                   (dict(out=None, o8=V(ROWS, H * 128, DT_I8)), ARG), (dict(out=None, os=V(ROWS, H, DT_F32)), ARG),
                   (dict(out=V(ROWS - 1, H * 128, DT_F32)), VIEW), (dict(out=V(ROWS, H * 128 - 1, DT_F32)), VIEW),
                   (dict(out=V(ROWS, H * 128, DT_I8)), DTYPE), (dict(hd=64), UNSUPPORTED),
                   (dict(out=C.byref(_lib.View(_ADDR + 2, H * 512, 4, ROWS, H * 128, DT_F32))), VIEW),
                   (dict(out=None, o8=V(ROWS, H * 128, DT_I8), os=V(ROWS, H - 1, DT_F32)), VIEW)]:
        assert attend(lib, **kw) == rc, kw
    assert pages(lib, hd=64) == UNSUPPORTED


@pytest.mark.parametrize("call", [pages, select])
def test_ids_refused(lib, call):
    for kw, rc in [(dict(ids=None), ARG), (dict(ids=V(ROWS, KV * 3, DT_F32)), DTYPE), (dict(ids=V(ROWS, KV * 3 - 1, DT_I32)), VIEW),
                   (dict(ids=V(ROWS - 1, KV * 3, DT_I32)), VIEW), (dict(n_sel=0), RANGE), (dict(n_sel=65537), RANGE), (dict(n_sel=4), VIEW),
                   (dict(ids=C.byref(_lib.View(_ADDR + 1, KV * 12, 4, ROWS, KV * 3, DT_I32))), VIEW)]:
        assert call(lib, **kw) == rc, kw


def test_heads_refused(lib):
    wide = pool(row_bytes=513 * 128, page_bytes=32 * 513 * 128, scale_row_bytes=513 * 4, scale_page_bytes=32 * 513 * 4)
    assert bounds(lib, kv=wide, kvh=513, b=V(16 * 513, 256, DT_I8), bs=V(16, 513, DT_F32)) == ARG
    assert attend(lib, q8=V(ROWS, 513 * 128, DT_I8), qs=V(ROWS, 513, DT_F32), out=V(ROWS, 513 * 128, DT_F32), heads=513, kvh=513, kv=wide) == ARG


@pytest.mark.parametrize("call", ["select", "bounds"])
def test_bounds_refused(lib, call):
    for b, bs, rc in [(V(31, 256, DT_I8), V(16, 2, DT_F32), VIEW), (V(32, 255, DT_I8), V(16, 2, DT_F32), VIEW),
                      (V(32, 256, DT_I8), V(15, 2, DT_F32), VIEW), (V(32, 256, DT_I8), V(16, 1, DT_F32), VIEW),
                      (V(32, 256, DT_F32), V(16, 2, DT_F32), DTYPE), (None, V(16, 2, DT_F32), ARG), (V(32, 256, DT_I8), None, ARG),
                      (V(32, 256, DT_I8), V(16, 2, DT_F32, row_bytes=16, col_bytes=8), VIEW)]:
        assert (select(lib, bounds=b, bscale=bs) if call == "select" else bounds(lib, b=b, bs=bs)) == rc
    assert select(lib, bounds=V(32, 256, DT_I8, row_bytes=264)) == VIEW
    assert select(lib, heads=34) == VIEW and select(lib, q8=V(ROWS, 34 * 128, DT_I8), qs=V(ROWS, 34, DT_F32), heads=34) == UNSUPPORTED


def workspace(lib, rows=ROWS, n_sel=0, heads=H, kvh=KV, pt=32, **kw):
    n = C.c_uint64(77)
    rc = lib.q3_seqs_workspace(seqs(**kw), rows, pt, heads, kvh, n_sel, C.byref(n))
    return rc, n.value


def test_workspace(lib):
    big = dict(ld_table=4096, max_kv=131072, max_rows=1)
    for kw in (dict(), dict(n_sel=3), dict(rows=64, **big), dict(rows=64, n_sel=64, **big), dict(rows=0, n_sel=3)):
        rc, n = workspace(lib, **kw)
        assert rc == OK and n < 1 << 32
    # more rows, keys or pages never need less, and a call with less than it needs is refused
    assert workspace(lib, rows=64, **big)[1] >= workspace(lib, rows=32, **big)[1]
    rc, n = workspace(lib, n_sel=3, **big)
    assert n >= 4 * ROWS * KV * 4096
    assert select(lib, s=seqs(**big), n=4 * ROWS * KV * 4096 - 1) == ARG
    assert select(lib, s=seqs(**big), ws=None, n=n) == ARG and select(lib, s=seqs(**big), ws=_ADDR + 4, n=n) == ARG
    for kw, want in [(dict(heads=0), ARG), (dict(kvh=0), ARG), (dict(heads=3), ARG), (dict(pt=0), ARG), (dict(rows=(1 << 30) + 1), RANGE),
                     (dict(n_sel=65537), RANGE), (dict(n_seq=65536), RANGE)]:
        assert workspace(lib, **kw)[0] == want, kw
    assert lib.q3_seqs_workspace(None, 1, 32, 4, 2, 0, C.byref(C.c_uint64())) == ARG
    assert lib.q3_seqs_workspace(seqs(), 1, 32, 4, 2, 0, None) == ARG


def test_unsupported_as_silent(lib):
    lib.q3_set_silent_unsupported(1)
    try:
        assert attend(lib, hd=64) == OK and append(lib, rot=63) == OK and bounds(lib, kv=pool(page_tokens=40)) == OK
        assert attend(lib, heads=3) == ARG
    finally:
        lib.q3_set_silent_unsupported(0)


# ---- rotary tables ---------------------------------------------------------------


def test_rope_tables_plain():
    cos, sin = rope_tables(300, 64, theta=1e4)
    f = 1e4 ** (-np.arange(32) / 32)
    a = np.arange(300)[:, None] * f
    assert cos.dtype == np.float32 and cos.shape == sin.shape == (300, 32)
    # one rounding to f32 of values up to 1 (half a step: 2^-25 below 1, 2^-24 at most)
    assert np.abs(cos - np.cos(a)).max() <= 2.0 ** -24 and np.abs(sin - np.sin(a)).max() <= 2.0 ** -24


def test_rope_tables_scaled():
    plain = rope_tables(4096, 128)
    cos, sin = rope_tables(4096, 128, scaling="linear", factor=4.0)
    assert np.array_equal(cos[::4], plain[0][:1024]) and np.array_equal(sin[::4], plain[1][:1024])
    cos, sin = rope_tables(4096, 128, scaling="ntk", factor=4.0)
    assert np.allclose(cos[:, 0], plain[0][:, 0], rtol=0, atol=2.0 ** -23)  # the fastest dimension as it was
    assert np.allclose(cos[4::4, -1], plain[0][1:1024, -1], rtol=0, atol=2.0 ** -22)  # the slowest by the factor
    cos, sin = rope_tables(4096, 128, scaling="yarn", factor=4.0, original=1024, attention_factor=1.0)
    turns = 1024 * 1e6 ** (-np.arange(64) / 64) / (2 * math.pi)
    fast, slow = turns > 32 * 1.3, turns < 1 / 1.3
    assert fast.any() and slow.any()
    assert np.array_equal(cos[:, fast], plain[0][:, fast])
    assert np.allclose(cos[4::4, slow], plain[0][1:1024, slow], rtol=0, atol=2.0 ** -22)
    scaled = rope_tables(64, 128, scaling="yarn", factor=4.0, original=1024)
    assert abs(scaled[0][0, 0] - (0.1 * math.log(4.0) + 1)) <= 2.0 ** -23
    assert rope_tables(0, 2)[0].shape == (0, 1)


def test_rope_tables_refused():
    for kw in (dict(rot_dim=0), dict(rot_dim=130), dict(rot_dim=7), dict(scaling="other"), dict(factor=0.5, scaling="linear"),
               dict(scaling="yarn", factor=2.0), dict(scaling="ntk", rot_dim=2, factor=2.0), dict(theta=0.0), dict(positions=-1)):
        with pytest.raises(ValueError):
            rope_tables(**{"positions": 8, **kw})
