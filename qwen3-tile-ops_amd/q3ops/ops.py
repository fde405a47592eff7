"""Python mirror of the reference operator surface (kernels/*.h) over the C
ABI.  Arguments are torch tensors on the GPU (or None where the reference
passes nullptr); names, argument order and meaning follow the reference
signatures cited on each function.  Shapes follow the reference's
MatrixView conventions: 2-D row-major tensors, and [n][1] column vectors for
per-row scales and norm gains (a 1-D tensor is taken as [n][1]).

Every call enqueues work on torch's current stream and raises Q3Error on a
non-zero status.  There is no fallback path: the HIP library must be built.
"""
from __future__ import annotations

import ctypes as C
from ctypes import byref

import torch

from ._lib import DT_F32, DT_I8, DT_I32, LM_ARGMAX, PagedKV, Q3Error, Seqs, View, check, lib

# element size and dtype code of the view dtypes
_DT = {torch.int8: (1, DT_I8), torch.float32: (4, DT_F32), torch.int32: (4, DT_I32)}


def view(t: torch.Tensor | None):
    """MatrixView of a tensor (kernels/matrix.h:27-34); None -> NULL.

    Each tensor attribute is read once: an operator makes up to a dozen views,
    and with two reads of most attributes they were most of a small call's
    host time (a one-row projection 11.7 us a call on the host)."""
    if t is None:
        return None
    known = _DT.get(t.dtype)
    if known is None:
        raise TypeError(f"unsupported dtype {t.dtype}")
    if not t.is_cuda:
        raise ValueError("operator views must point at device memory")
    es, code = known
    stride = t.stride()
    if len(stride) == 1:
        if stride[0] != 1:
            raise ValueError("1-D views must be contiguous")
        return byref(View(t.data_ptr(), es, es, t.shape[0], 1, code))
    if len(stride) != 2 or stride[1] != 1:
        raise ValueError("views must be 2-D with dense columns")
    rows, cols = t.shape
    return byref(View(t.data_ptr(), (stride[0] if rows > 1 else cols) * es, es, rows, cols, code))


def _stream(stream=None) -> int:
    """The hipStream_t of the stream, or of the current device's current one
    (read as the raw handle: a Stream object costs a microsecond)."""
    if stream is not None:
        return stream.cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _raw_stream(device: int) -> int:
    """torch.cuda.current_stream(device).cuda_stream, without the object where
    this torch has the raw getter."""
    get = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return get(device) if get else torch.cuda.current_stream(device).cuda_stream


def paged_kv(k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor,
             table: torch.Tensor, page_tokens: int = 32) -> PagedKV:
    """kernels/kv_pages.h:13-24.  k/v: [pages, page_tokens, kv_dim] int8,
    ks/vs: [pages, page_tokens, kv_heads] f32, table: int16/uint16-compatible
    logical->physical map on the device.

    The returned struct holds only device addresses, so it also keeps the
    five tensors alive (a freed table would be reallocated under the
    kernel's feet).  Every table entry is checked against the page count,
    because the C ABI, like the reference PagedKV, carries no page count."""
    for t in (k, v, ks, vs):
        assert t.is_cuda and t.is_contiguous()
    assert k.dtype == torch.int8 and v.dtype == torch.int8
    assert ks.dtype == torch.float32 and vs.dtype == torch.float32
    assert table.dtype in (torch.int16, torch.uint16) and table.is_cuda and table.is_contiguous()
    n_pages = k.shape[0]
    assert v.shape[0] == n_pages and ks.shape[0] == n_pages and vs.shape[0] == n_pages
    tab = table.cpu().numpy().view("uint16")
    if tab.size and int(tab.max()) >= n_pages:
        raise ValueError(f"page table entry {int(tab.max())} >= {n_pages} pages")
    kv_dim = k.shape[-1]
    kv_heads = ks.shape[-1]
    kv = PagedKV(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(),
                 page_tokens, page_tokens * kv_dim, kv_dim, page_tokens * kv_heads * 4,
                 kv_heads * 4)
    kv._keep = (k, v, ks, vs, table)
    kv.n_pages = n_pages
    kv.n_logical = table.numel()
    return kv


def _check_tokens(kv: PagedKV, end_token: int) -> None:
    n_logical = getattr(kv, "n_logical", None)
    if n_logical is not None and end_token > n_logical * kv.page_tokens:
        raise ValueError(f"token {end_token - 1} is beyond the page table "
                         f"({n_logical} pages of {kv.page_tokens})")


def embedding_rmsnorm_rows(table, scale, ids, tmp, w, out, inv, stream=None):
    """kernels/embedding.h:99-168."""
    check(lib().q3_embedding_rmsnorm_rows(view(table), view(scale), view(ids), view(tmp),
                                          view(w), view(out), C.c_float(inv), _stream(stream)),
          "embedding_rmsnorm_rows")


def rmsnorm_rows(x, w, out, inv, stream=None):
    """kernels/rmsnorm.h:34-81."""
    check(lib().q3_rmsnorm_rows(view(x), view(w), view(out), C.c_float(inv), _stream(stream)),
          "rmsnorm_rows")


def quant_rows_heads(x, qi8, scale, group_cols, stream=None):
    """kernels/quant.h:89-138."""
    check(lib().q3_quant_rows_heads(view(x), view(qi8), view(scale), group_cols,
                                    _stream(stream)), "quant_rows_heads")


def gemm_nt_group_store(a, a_scale, b, b_scale, out, group_k=128, add=None, q8=None, qs=None,
                        nw=None, cos=None, sin=None, inv_hd=0.0, stream=None):
    """kernels/group_gemm.h:27-222."""
    check(lib().q3_gemm_nt_group_store(view(a), view(a_scale), view(b), view(b_scale),
                                       view(out), group_k, view(add), view(q8), view(qs),
                                       view(nw), view(cos), view(sin), C.c_float(inv_hd),
                                       _stream(stream)), "gemm_nt_group_store")


def gemm_nt_group_kv_paged(a, a_scale, b, b_scale, group_k, kv: PagedKV, pos0, is_v, nw=None,
                           cos=None, sin=None, inv_hd=0.0, stream=None):
    """K/V epilogues of gemm_nt_group_store writing page slots
    (main_big.cpp:185-209)."""
    _check_tokens(kv, pos0 + a.shape[0])
    check(lib().q3_gemm_nt_group_kv_paged(view(a), view(a_scale), view(b), view(b_scale),
                                          group_k, C.byref(kv), pos0, int(is_v), view(nw),
                                          view(cos), view(sin), C.c_float(inv_hd),
                                          _stream(stream)), "gemm_nt_group_kv_paged")


def norm_rope_quant_heads(x, w, cos, sin, q8, scale, heads, inv_hd, do_rope=True, stream=None):
    """kernels/norm_rope_quant.h:88-111."""
    check(lib().q3_norm_rope_quant_heads(view(x), view(w), view(cos), view(sin), view(q8),
                                         view(scale), heads, C.c_float(inv_hd), int(do_rope),
                                         _stream(stream)), "norm_rope_quant_heads")


def attention_heads_gqa_tokscale_paged(q8, q_scale, kv: PagedKV, kv_len, o8, os, heads,
                                       kv_heads, head_dim, causal, qk_scale, stream=None):
    """kernels/attention_gqa.h:549-572."""
    _check_tokens(kv, kv_len)
    check(lib().q3_attention_heads_gqa_tokscale_paged(view(q8), view(q_scale), C.byref(kv),
                                                      kv_len, view(o8), view(os), heads,
                                                      kv_heads, head_dim, int(causal),
                                                      C.c_float(qk_scale), _stream(stream)),
          "attention_heads_gqa_tokscale_paged")


def gemm_gate_up_swiglu_quant(a, a_scale, wg, wgs, wu, wus, s8, ss, group_k=256, stream=None):
    """kernels/swiglu_quant.h:164-255."""
    check(lib().q3_gemm_gate_up_swiglu_quant(view(a), view(a_scale), view(wg), view(wgs),
                                             view(wu), view(wus), view(s8), view(ss), group_k,
                                             _stream(stream)), "gemm_gate_up_swiglu_quant")


def gemm_nt_group_argmax(a, a_scale, b, b_scale, best, bidx, group_k=128, stream=None):
    """kernels/lm_argmax.h:72-182 (best/bidx are read and updated)."""
    check(lib().q3_gemm_nt_group_argmax(view(a), view(a_scale), view(b), view(b_scale),
                                        view(best), view(bidx), group_k, _stream(stream)),
          "gemm_nt_group_argmax")


def gemm_nt_group_argmax_noalloc(a, a_scale, b, b_scale, best, bidx, group_k=128, stream=None):
    """gemm_nt_group_argmax with the library's fixed device key array instead
    of an allocated workspace (no reference counterpart; for callers that
    cannot allocate).  Calls that overlap on one GPU race."""
    check(lib().q3_gemm_nt_group_argmax_noalloc(view(a), view(a_scale), view(b), view(b_scale),
                                                view(best), view(bidx), group_k,
                                                _stream(stream)),
          "gemm_nt_group_argmax_noalloc")


def argmax_logits(logits, out_id, stream=None):
    """main_big.cpp:300-322 (out_id: int32 device tensor, element 0)."""
    check(lib().q3_argmax_logits(view(logits), C.c_void_p(out_id.data_ptr()), _stream(stream)),
          "argmax_logits")


# ---- batches of sequences over one paged cache ------------------------------


MAX_ROWS = 1 << 21  # of a call on a batch of sequences


def kv_pool(k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor) -> PagedKV:
    """The pool of K/V pages that the batch operators below share: k/v
    [pages, page_tokens, kv_heads * 128] int8, ks/vs [pages, page_tokens,
    kv_heads] f32, contiguous.  Unlike paged_kv it holds no table (each call's
    tables come with its sequences), so making it reads nothing back."""
    if k.dim() != 3 or ks.dim() != 3 or v.shape != k.shape or vs.shape != ks.shape or ks.shape[:2] != k.shape[:2]:
        raise ValueError("k/v are [pages, page_tokens, kv_heads * 128], ks/vs [pages, page_tokens, kv_heads]")
    n_pages, page_tokens, kv_dim = k.shape
    kv_heads = ks.shape[2]
    if kv_dim != kv_heads * 128:
        raise ValueError(f"rows of {kv_dim} columns for {kv_heads} heads of 128")
    for t, dt in ((k, torch.int8), (v, torch.int8), (ks, torch.float32), (vs, torch.float32)):
        if t.dtype != dt:
            raise TypeError(f"unsupported dtype {t.dtype}")
        if not t.is_contiguous():
            raise ValueError("the pool's tensors must be contiguous")
        _on_device(t, k)
    kv = PagedKV(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), None, page_tokens,
                 page_tokens * kv_dim, kv_dim, page_tokens * kv_heads * 4, kv_heads * 4)
    kv._keep = (k, v, ks, vs)
    kv.n_pages, kv.kv_heads, kv.device = n_pages, kv_heads, k.device
    return kv


def sequences(pool: PagedKV, tables, row_start, kv_len, max_rows: int, max_kv: int) -> Seqs:
    """The batch of one call (q3_seqs): tables [n_seq, pages] int16/uint16
    logical -> physical pages, row_start [n_seq + 1] and kv_len [n_seq] int32, on
    the pool's device; max_rows and max_kv are the host's limits of the new rows
    and of the cached tokens of a sequence.  The arrays' contents may change
    between calls (or replays of a captured one) within these limits."""
    if tables.dtype not in (torch.int16, torch.uint16) or row_start.dtype != torch.int32 or kv_len.dtype != torch.int32:
        raise TypeError("tables are int16 or uint16, row_start and kv_len int32")
    n_seq = kv_len.shape[0]
    if kv_len.dim() != 1 or tables.dim() != 2 or tables.shape[0] != n_seq or row_start.shape != (n_seq + 1,):
        raise ValueError("tables are [n_seq, pages], row_start [n_seq + 1], kv_len [n_seq]")
    index = pool.device.index
    for t in (tables, row_start, kv_len):
        if not t.is_contiguous():
            raise ValueError("tables, row_start and kv_len must be contiguous")
        if t.get_device() != index:
            _on_device(t, pool)
    s = Seqs(row_start.data_ptr(), kv_len.data_ptr(), tables.data_ptr(), n_seq, tables.shape[1],
             pool.n_pages, max_rows, max_kv)
    s._keep = (tables, row_start, kv_len)
    s.index = index
    return s


def _on_device(t, like) -> None:
    if not t.is_cuda:
        raise ValueError("operator views must point at device memory")
    if t.device != like.device:
        raise ValueError(f"tensors on {t.device} and {like.device}")


def _views(pool: PagedKV, tensors) -> list:
    """view() of each tensor, all on the pool's device (one loop over them: at one
    row the wrapper is most of a call's time, and a call per tensor half of that)."""
    index, out = pool.device.index, []
    for t in tensors:
        if t is None:
            out.append(None)
            continue
        if t.get_device() != index:
            raise ValueError("operator views must point at device memory" if not t.is_cuda
                             else f"tensors on {t.device} and {pool.device}")
        known = _DT.get(t.dtype)
        stride = t.stride()
        if known is None or len(stride) != 2 or stride[1] != 1:
            out.append(view(t))  # a vector, or an error
            continue
        es, code = known
        rows, cols = t.shape
        out.append(byref(View(t.data_ptr(), (stride[0] if rows > 1 else cols) * es, es, rows, cols, code)))
    return out


def _heads(rows) -> int:
    heads, rest = divmod(rows.shape[1], 128)
    if rest:
        raise ValueError(f"rows of {rows.shape[1]} columns are not heads of 128")
    return heads


def _launch_stream(pool: PagedKV, seqs: Seqs, stream) -> int:
    """The stream of a call on the pool's device, which has to be the current one
    (kernels launch there).  Sequences of another pool do as well (a layer's), if
    their tables' pages are this one's too."""
    dev = pool.device
    if seqs.n_pages > pool.n_pages or seqs.index != dev.index:
        raise ValueError(f"sequences over {seqs.n_pages} pages on cuda:{seqs.index} for a pool of {pool.n_pages} on {dev}")
    if dev.index != torch.cuda.current_device():
        raise ValueError(f"the pool is on {dev}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is None:
        return _raw_stream(dev.index)
    if stream.device != dev:
        raise ValueError(f"a stream of {stream.device} for a pool on {dev}")
    return stream.cuda_stream


def rope_append_paged(q, k, v, pool: PagedKV, seqs: Seqs, q8=None, qs=None, nwq=None, nwk=None, inv_hd=1 / 128,
                      cos=None, sin=None, rot_dim=128, interleaved=False, stream=None):
    """q3_rope_append_paged: new Q/K/V rows (f32 [rows, heads * 128]) of every
    sequence, normed (gains nwq / nwk), rotated at their positions (cos / sin
    [position, rot_dim / 2], e.g. rope_tables'; None: not rotated), quantised; K
    and V into their pages, Q into q8 / qs (q None: K and V alone)."""
    vq, vk, vv, vnq, vnk, vc, vs, v8, vqs = _views(pool, (q, k, v, nwq, nwk, cos, sin, q8, qs))
    check(lib().q3_rope_append_paged(vq, vk, vv, vnq, vnk, inv_hd, vc, vs, rot_dim if cos is not None else 0,
                                     int(interleaved), v8, vqs, byref(pool), byref(seqs),
                                     0 if q is None else _heads(q), pool.kv_heads,
                                     _launch_stream(pool, seqs, stream)), "rope_append_paged")


def page_bounds(pool: PagedKV, seqs: Seqs, bounds, bscale, rows: int | None = None, stream=None):
    """q3_page_bounds: channel bounds (int8 [pages * kv_heads, 256], least then
    largest; f32 [pages, kv_heads]) of the pages that the sequences' new rows lie
    in (rows: the call's row count; without it row_start is taken as it is)."""
    rows = MAX_ROWS if rows is None else rows
    vb, vs = _views(pool, (bounds, bscale))
    check(lib().q3_page_bounds(byref(pool), byref(seqs), rows, pool.kv_heads, vb, vs, _launch_stream(pool, seqs, stream)),
          "page_bounds")


def seqs_workspace_bytes(pool: PagedKV, seqs: Seqs, rows: int, heads: int, n_sel: int = 0) -> int:
    """q3_seqs_workspace: bytes for attention_varlen_paged and, with n_sel,
    select_pages and attention_pages on these sizes, and on any smaller ones."""
    n = C.c_uint64()
    check(lib().q3_seqs_workspace(byref(seqs), rows, pool.page_tokens, heads, pool.kv_heads, n_sel, byref(n)),
          "seqs_workspace")
    return n.value


def _workspace_on(ws, stream, pool, seqs, q8, n_sel):
    """The caller's workspace tensor, or a new one (torch's allocator hands its
    memory out again in the order of the current stream)."""
    if ws is None:
        n = seqs_workspace_bytes(pool, seqs, q8.shape[0], _heads(q8), n_sel)
        if n == 0:
            return None, None, 0
        if stream is not None and stream != torch.cuda.current_stream(pool.device):
            raise ValueError("a call on a stream that is not the current one needs its workspace given")
        ws = torch.empty(n, dtype=torch.uint8, device=pool.device)
        return ws, ws.data_ptr(), n
    if not ws.is_contiguous() or ws.device != pool.device:
        raise ValueError("the workspace must be contiguous and on the pool's device")
    return ws, ws.data_ptr(), ws.numel() * ws.element_size()


def attention_varlen_paged(q8, q_scale, pool: PagedKV, seqs: Seqs, out=None, o8=None, os=None, causal=True,
                           qk_scale=128 ** -0.5, workspace=None, stream=None):
    """q3_attention_varlen_paged: attention of every sequence's rows over its
    cached keys; the result in f32 (out) or int8 with a scale per head (o8, os).
    workspace: a device tensor of seqs_workspace_bytes, needed on a stream that
    is not the current one; otherwise one is allocated."""
    vq, vs, vo, v8, vos = _views(pool, (q8, q_scale, out, o8, os))
    st = _launch_stream(pool, seqs, stream)
    keep, ws, n = _workspace_on(workspace, stream, pool, seqs, q8, 0)
    check(lib().q3_attention_varlen_paged(vq, vs, byref(pool), byref(seqs), vo, v8, vos, _heads(q8),
                                          pool.kv_heads, 128, int(causal), qk_scale, ws, n, st),
          "attention_varlen_paged")


def select_pages(q8, q_scale, pool: PagedKV, seqs: Seqs, bounds, bscale, ids, n_sel, workspace=None, stream=None):
    """q3_select_pages: the n_sel pages of each row and KV head with the largest
    bounds of a score, into ids (int32 [rows, kv_heads * n_sel])."""
    vq, vs, vb, vbs, vi = _views(pool, (q8, q_scale, bounds, bscale, ids))
    st = _launch_stream(pool, seqs, stream)
    keep, ws, n = _workspace_on(workspace, stream, pool, seqs, q8, n_sel)
    check(lib().q3_select_pages(vq, vs, byref(pool), byref(seqs), vb, vbs, vi, n_sel, _heads(q8),
                                pool.kv_heads, ws, n, st), "select_pages")


def attention_pages(q8, q_scale, pool: PagedKV, seqs: Seqs, ids, n_sel, out=None, o8=None, os=None,
                    qk_scale=128 ** -0.5, workspace=None, stream=None):
    """q3_attention_pages: attention_varlen_paged over the keys of each row's
    listed pages (select_pages' ids, or the caller's own)."""
    vq, vs, vi, vo, v8, vos = _views(pool, (q8, q_scale, ids, out, o8, os))
    st = _launch_stream(pool, seqs, stream)
    keep, ws, n = _workspace_on(workspace, stream, pool, seqs, q8, n_sel)
    check(lib().q3_attention_pages(vq, vs, byref(pool), byref(seqs), vi, n_sel, vo, v8, vos, _heads(q8),
                                   pool.kv_heads, 128, qk_scale, ws, n, st), "attention_pages")


__all__ = ["Q3Error", "view", "paged_kv", "embedding_rmsnorm_rows", "rmsnorm_rows", "quant_rows_heads",
           "gemm_nt_group_store", "gemm_nt_group_kv_paged", "norm_rope_quant_heads",
           "attention_heads_gqa_tokscale_paged", "gemm_gate_up_swiglu_quant",
           "gemm_nt_group_argmax", "gemm_nt_group_argmax_noalloc", "argmax_logits", "LM_ARGMAX",
           "kv_pool", "sequences", "rope_append_paged", "page_bounds", "seqs_workspace_bytes",
           "attention_varlen_paged", "select_pages", "attention_pages"]
