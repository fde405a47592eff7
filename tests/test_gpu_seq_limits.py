"""The batch operators at the limits of their counts, and workspaces sized for them."""
from __future__ import annotations

import numpy as np
import pytest

from seqref import F, Batch, attend, attend_bound, queries
from test_gpu_seq_ops import QK, dev, on_device, ops, torch

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
