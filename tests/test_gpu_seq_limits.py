"""The batch operators at the limits of their counts, and workspaces sized for them."""
from __future__ import annotations

import numpy as np
import pytest

from seqref import F, Batch, attend, attend_bound, queries
from test_gpu_seq_ops import QK, check_attention, dev, on_device, ops, torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 3])
def test_attention_a_billion_keys(cuda, rows):
    """A sequence near max_kv's limit of 2^30, of whose pages only the first and the last lie
    in the pool, beside short ones: with three tiles of columns it takes 21 of the 64 splits
    launched, whose starts would lie at up to three times its length."""
    page, n, tail = 1 << 16, 24, 40000
    b = Batch([(rows, page + tail - rows)], 1, page, seed=7, spare_pages=0)
    q8, qs = queries(b.rng, n * rows, 16)
    kv_len = np.full(n, rows, np.int32)
    last = 10 ** 9 // page
    kv_len[0] = last * page + tail
    tables = np.full((n, (1 << 30) // page), 65535, np.uint16)
    tables[0, [0, last]] = b.tables[0]
    pool, _ = on_device(b)
    seqs = ops.sequences(pool, dev(tables), dev((rows * np.arange(n + 1)).astype(np.int32)), dev(kv_len), rows, 1 << 30)
    out = torch.full((n * rows, 16 * 128), 7.5, device="cuda")
    ops.attention_varlen_paged(dev(q8), dev(qs), pool, seqs, out, qk_scale=QK)
    got = out.cpu().numpy()
    want, mag, top = attend(b, q8[:rows], qs[:rows], 16, QK)
    assert (np.abs(got[:rows] - want) <= attend_bound(mag, top, b.max_kv)).all()
    assert (got[rows:] == 0).all()  # of pages outside the pool


@pytest.mark.parametrize("heads,kv_heads,n_sel", [(16, 8, 0), (16, 8, 12), (16, 1, 9)])
def test_workspace_of_the_largest_counts(cuda, heads, kv_heads, n_sel):
    """One workspace, sized for a loop's largest counts, serves every smaller call; what lies
    behind it is left alone."""
    rng = np.random.default_rng(heads + n_sel)
    rows, n_seq, max_kv = 4096, 64, 8192
    b = Batch([(1, 600)] * 3 + [(8, 400)], kv_heads, 32, seed=9)
    b.ks[:], b.vs[:] = np.nan_to_num(b.ks, nan=0.02), np.nan_to_num(b.vs, nan=0.02)
    pool, _ = on_device(b)
    wide = np.full((n_seq, max_kv // 32), 65535, np.uint16)
    for i in range(n_seq):
        wide[i, :b.tables.shape[1]] = b.tables[i % 4]
    tables = dev(wide)
    q8, qs = (dev(t) for t in queries(rng, rows, heads))
    ids = torch.arange(n_sel, dtype=torch.int32, device="cuda").repeat(rows, kv_heads) if n_sel else None
    most = ops.sequences(pool, tables, *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (n_seq + 1, n_seq)), rows, max_kv)
    n = ops.seqs_workspace_bytes(pool, most, rows, heads, n_sel)
    ws = torch.full((n + 4096,), 77, dtype=torch.uint8, device="cuda")
    out = torch.empty((rows, heads * 128), device="cuda")
    for r, s, mr, kv in [(8, 1, 8, 600), (64, 64, 1, 608), (64, 64, 1, 8192), (27, 27, 1, 1792), (200, 20, 100, 1793), (300, 3, 300, 700), (1024, 1, 1024, 8192),
                         (1024, 12, 1024, 768), (2048, 1, 2048, 700), (3000, 60, 48, 900), (4096, 1, 4096, 8192), (4096, 64, 64, 608)]:
        starts = np.minimum(np.arange(s + 1) * mr, r).astype(np.int32)
        kv_len = np.full(s, min(kv, 600), np.int32)
        seqs = ops.sequences(pool, tables[:s], dev(starts), dev(kv_len), mr, kv)
        got, want = out[:r].fill_(7.5), torch.full((r, heads * 128), 7.5, device="cuda")
        for o, w in ((got, ws[:n]), (want, None)):
            if n_sel:
                ops.attention_pages(q8[:r], qs[:r], pool, seqs, ids[:r], n_sel, o, qk_scale=QK, workspace=w)
            else:
                ops.attention_varlen_paged(q8[:r], qs[:r], pool, seqs, o, qk_scale=QK, workspace=w)
        assert torch.equal(got, want) and bool(torch.isfinite(got).all()), (r, s, mr, kv)
        assert (ws[n:] == 77).all(), (r, s, mr, kv)


@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (6, 2)])
def test_unequal_chunks_of_a_small_call(cuda, heads, kv_heads):
    """16-column tiles alone, split, of sequences far from equal: the partial results lie by
    row, not by the longest's columns of each."""
    b = Batch([(200, 400), (1, 900), (0, 30), (3, 500), (60, 0), (1, 0), (2, 1200)], kv_heads, 32, seed=heads, before=2, behind=5)
    assert b.rows * heads * b.max_kv <= 12 << 20
    pool, seqs = on_device(b)
    assert 0 < ops.seqs_workspace_bytes(pool, seqs, b.rows, heads) <= b.rows * heads * 5 * 520  # of 1201 keys in 256 or more
    check_attention(b, heads)
