"""q3_seqs_workspace without a GPU: a size for some counts serves all smaller ones."""
from __future__ import annotations

import ctypes as C
import random

import pytest

from q3ops import _lib

COUNTS = ("rows", "n_seq", "max_rows", "max_kv", "n_sel")


def need(heads, kv_heads, page, rows, n_seq, max_rows, max_kv, n_sel):
    s = _lib.Seqs(None, None, None, n_seq, -(-max_kv // page), 16, max_rows, max_kv)
    n = C.c_uint64()
    assert _lib.lib().q3_seqs_workspace(C.byref(s), rows, page, heads, kv_heads, n_sel, C.byref(n)) == 0
    return n.value


SIZES = {"rows": (0, 1, 2, 7, 16, 17, 64, 100, 256, 1000, 1024, 2048, 4096, 8192, 1 << 17), "n_seq": (0, 1, 2, 3, 20, 27, 64, 96, 97, 192, 200, 768, 769, 4096),
         "max_rows": (0, 1, 2, 3, 16, 24, 25, 48, 100, 1024, 4096, 8192), "max_kv": (0, 1, 256, 257, 384, 385, 512, 543, 1792, 1793, 4096, 8192, 131072, 1 << 30),
         "n_sel": (0, 1, 4, 8, 9, 64, 255, 300, 4096)}


@pytest.mark.parametrize("heads,kv_heads,page", [(16, 8, 32), (16, 1, 32), (64, 8, 64), (33, 1, 96), (20, 4, 256), (8, 8, 32)])
def test_never_less_for_larger_counts(heads, kv_heads, page):
    rng = random.Random(heads * page)
    for _ in range(4000):
        at = {k: rng.choice(v) for k, v in SIZES.items()}
        more = {k: rng.choice([x for x in SIZES[k] if x >= at[k]]) for k in COUNTS}
        small, large = need(heads, kv_heads, page, **at), need(heads, kv_heads, page, **more)
        assert small <= large, (at, more)
        scores = 4 * more["rows"] * kv_heads * -(-more["max_kv"] // page) if more["n_sel"] else 0
        assert large <= max(154 << 20, scores)


def test_sizes_of_a_serving_loop():
    """Counts whose own calls need more than larger ones did."""
    of = lambda **kw: need(16, 8, 32, **{"rows": 8192, "n_seq": 1, "max_rows": 8192, "max_kv": 8192, "n_sel": 0, **kw})  # noqa: E731
    assert of(rows=4096, max_rows=4096) <= of() and of(rows=1024, max_rows=1024) <= of()
    decode = lambda n, kv: of(rows=n, n_seq=n, max_rows=1, max_kv=kv)  # noqa: E731
    assert 0 < decode(64, 4096) <= decode(200, 4096) <= 2 << 20  # no more than a split's results for each workgroup
    assert decode(27, 1792) <= decode(27, 1793)
    assert decode(1, 256) == 0 and decode(1, 257) > 0
