// C ABI of the operators on batches of sequences (include/q3ops.h): argument
// checks and dispatch.  Row starts, lengths and tables lie on the device and are
// never read here; the kernels clamp what they read (q3_seq.h).
#include "q3_check.h"
#include "q3_seq.h"
#include "q3ops.h"

namespace {

using q3::check_scales;
using q3::check_vec;
using q3::check_view;
using q3::hip_status;
using q3::ld;
using q3::unsupported;

constexpr uint32_t kMaxTokens = 1u << 30;  // positions are 32-bit on the device
constexpr uint32_t kMaxRows = 1u << 21;    // rows x heads, and twice that, are 32-bit too
constexpr int kMaxHeads = 512;
constexpr uint32_t kMaxSeqs = 4096;  // a 128-column tile's workgroup looks through them all

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The pool and the sequences of a call over `rows` rows.
int seq_common(const q3_paged_kv *kv, const q3_seqs *q, uint32_t rows, int kv_heads, q3::Pool &p, q3::Seqs &s) {
  if (!kv || !kv->k || !kv->v || !kv->ks || !kv->vs || !q) return Q3_ERR_ARG;
  if (kv_heads <= 0 || kv_heads > kMaxHeads) return Q3_ERR_ARG;
  if (kv->page_tokens == 0 || kv->page_tokens % 32 != 0) return Q3_ERR_UNSUPPORTED;
  const uint64_t pt = kv->page_tokens;
  if (kv->page_bytes < pt * kv->row_bytes || kv->scale_page_bytes < pt * kv->scale_row_bytes) return Q3_ERR_VIEW;
  if (kv->row_bytes % 16 || kv->page_bytes % 16 || kv->scale_row_bytes % 4 || kv->scale_page_bytes % 4) return Q3_ERR_VIEW;
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->ks, 4) || !aligned(kv->vs, 4)) return Q3_ERR_VIEW;
  if (kv->row_bytes / 128 < static_cast<uint32_t>(kv_heads) || kv->scale_row_bytes / 4 < static_cast<uint32_t>(kv_heads))
    return Q3_ERR_VIEW;
  if (q->n_seq && (!q->row_start || !q->kv_len || !q->tables)) return Q3_ERR_ARG;
  if (!aligned(q->row_start, 4) || !aligned(q->kv_len, 4) || !aligned(q->tables, 2)) return Q3_ERR_VIEW;
  if (q->n_seq > kMaxSeqs || rows > kMaxRows || q->max_kv > kMaxTokens || pt > kMaxTokens) return Q3_ERR_RANGE;
  if (q->max_kv > q->ld_table * pt) return Q3_ERR_RANGE;  // keys behind the table
  if (q->max_rows > rows && q->n_seq) return Q3_ERR_RANGE;
  p = {static_cast<int8_t *>(kv->k), static_cast<int8_t *>(kv->v), static_cast<float *>(kv->ks), static_cast<float *>(kv->vs),
       kv->page_bytes, kv->row_bytes, kv->scale_page_bytes / 4, kv->scale_row_bytes / 4,
       static_cast<int>(pt), static_cast<int>(q->n_pages < 65536 ? q->n_pages : 65536)};
  s = {q->row_start, q->kv_len, q->tables, q->ld_table, static_cast<int>(q->n_seq), static_cast<int>(rows),
       static_cast<int>(q->max_rows), static_cast<int>(q->max_kv)};
  return Q3_OK;
}

// Queries [rows][heads * 128] int8 with a scale per head.
int check_queries(const q3_view *q8, const q3_view *q_scale, int heads, int kv_heads) {
  Q3_TRY(check_view(q8, Q3_DT_I8));
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > kMaxHeads) return Q3_ERR_ARG;
  if (q8->cols < static_cast<uint32_t>(heads) * 128) return Q3_ERR_VIEW;
  if (q8->row_bytes % 16 || !aligned(q8->data, 16)) return Q3_ERR_VIEW;
  return check_scales(q_scale, q8->rows, static_cast<uint32_t>(heads));
}

// Where the attention's result goes: f32 rows, or int8 rows and their scales.
int check_out(const q3_view *out, const q3_view *o8, const q3_view *os, uint32_t rows, int heads, q3::SeqAttnArgs &a) {
  const uint32_t cols = static_cast<uint32_t>(heads) * 128;
  if (!out == !o8 || !o8 != !os) return Q3_ERR_ARG;  // one of the two forms
  if (out) {
    Q3_TRY(check_view(out, Q3_DT_F32));
    if (out->rows < rows || out->cols < cols || !aligned(out->data, 4)) return Q3_ERR_VIEW;
    a.out = static_cast<float *>(out->data);
    a.ldo = ld(out);
  } else {
    Q3_TRY(check_view(o8, Q3_DT_I8));
    if (o8->rows < rows || o8->cols < cols) return Q3_ERR_VIEW;
    Q3_TRY(check_scales(os, rows, static_cast<uint32_t>(heads)));
    a.o8 = static_cast<int8_t *>(o8->data);
    a.ldo8 = o8->row_bytes;
    a.os = static_cast<float *>(os->data);
    a.ldos = os->row_bytes / 4;
    a.os_col = os->col_bytes / 4;
  }
  return Q3_OK;
}

int attn_common(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs, const q3_view *out,
                const q3_view *o8, const q3_view *os, int heads, int kv_heads, int head_dim, float qk_scale, q3::SeqAttnArgs &a) {
  Q3_TRY(check_queries(q8, q_scale, heads, kv_heads));
  if (head_dim != 128) return Q3_ERR_UNSUPPORTED;
  Q3_TRY(seq_common(kv, seqs, q8->rows, kv_heads, a.pool, a.seqs));
  Q3_TRY(check_out(out, o8, os, q8->rows, heads, a));
  a.q8 = static_cast<const int8_t *>(q8->data);
  a.ldq = q8->row_bytes;
  a.qs = static_cast<const float *>(q_scale->data);
  a.ldqs = q_scale->row_bytes / 4;
  a.qs_col = q_scale->col_bytes / 4;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.qk_scale = qk_scale;
  return Q3_OK;
}

// ids [rows][kv_heads * n_sel] int32.
int check_ids(const q3_view *ids, uint32_t rows, int kv_heads, uint32_t n_sel) {
  Q3_TRY(check_view(ids, Q3_DT_I32));
  if (n_sel == 0 || n_sel > 65536) return Q3_ERR_RANGE;
  if (ids->rows < rows || ids->cols < static_cast<uint64_t>(kv_heads) * n_sel || !aligned(ids->data, 4)) return Q3_ERR_VIEW;
  return Q3_OK;
}

// Keys of a selection's scores: one row of them per (row, KV head).
int64_t score_ld(const q3_seqs *q, uint32_t page_tokens) { return (q->max_kv + int64_t(page_tokens) - 1) / page_tokens; }

int check_ws(const void *ws, uint64_t have, uint64_t need) {
  if (need == 0) return Q3_OK;
  return ws && aligned(ws, 16) && have >= need ? Q3_OK : Q3_ERR_ARG;
}

// Operators that a caller turned into silent no-ops on unsupported shapes.
int finish(int rc) { return rc == Q3_ERR_UNSUPPORTED ? unsupported() : rc; }

int append(const q3_view *q, const q3_view *k, const q3_view *v, const q3_view *nwq, const q3_view *nwk, float inv_hd,
           const q3_view *cos, const q3_view *sin, uint32_t rot_dim, int interleaved, const q3_view *q8, const q3_view *qs,
           const q3_paged_kv *kv, const q3_seqs *seqs, int heads, int kv_heads, void *stream) {
  q3::SeqAppendArgs a{};
  Q3_TRY(check_view(k, Q3_DT_F32));
  Q3_TRY(check_view(v, Q3_DT_F32));
  const uint32_t rows = k->rows;
  if (kv_heads <= 0 || kv_heads > kMaxHeads || heads < 0 || heads > kMaxHeads) return Q3_ERR_ARG;
  if (!q != (heads == 0) || !q != !q8 || !q8 != !qs || (!q && nwq)) return Q3_ERR_ARG;
  if (v->rows != rows || k->cols < kv_heads * 128u || v->cols < kv_heads * 128u) return Q3_ERR_VIEW;
  if (!aligned(k->data, 4) || !aligned(v->data, 4)) return Q3_ERR_VIEW;
  if (q) {
    Q3_TRY(check_view(q, Q3_DT_F32));
    Q3_TRY(check_view(q8, Q3_DT_I8));
    if (q->rows != rows || q8->rows < rows || q->cols < heads * 128u || q8->cols < heads * 128u) return Q3_ERR_VIEW;
    if (!aligned(q->data, 4) || !aligned(q8->data, 4) || q8->row_bytes % 4) return Q3_ERR_VIEW;
    Q3_TRY(check_scales(qs, rows, static_cast<uint32_t>(heads)));
    a.q = static_cast<const float *>(q->data);
    a.ldq = ld(q);
    a.q8 = static_cast<int8_t *>(q8->data);
    a.ldq8 = q8->row_bytes;
    a.qs = static_cast<float *>(qs->data);
    a.ldqs = qs->row_bytes / 4;
    a.qs_col = qs->col_bytes / 4;
  }
  if (nwq) {
    Q3_TRY(check_vec(nwq, 128, &a.nwq_stride));
    a.nwq = static_cast<const float *>(nwq->data);
  }
  if (nwk) {
    Q3_TRY(check_vec(nwk, 128, &a.nwk_stride));
    a.nwk = static_cast<const float *>(nwk->data);
  }
  Q3_TRY(seq_common(kv, seqs, rows, kv_heads, a.pool, a.seqs));
  if (!cos != !sin || !cos != (rot_dim == 0)) return Q3_ERR_ARG;
  if (rot_dim > 128 || rot_dim % 2) return Q3_ERR_UNSUPPORTED;
  if (cos) {
    Q3_TRY(check_view(cos, Q3_DT_F32));
    Q3_TRY(check_view(sin, Q3_DT_F32));
    if (cos->cols < rot_dim / 2 || sin->cols < rot_dim / 2 || cos->row_bytes != sin->row_bytes) return Q3_ERR_VIEW;
    if (cos->rows < seqs->max_kv || sin->rows < seqs->max_kv) return Q3_ERR_RANGE;  // positions without angles
    a.cos_t = static_cast<const float *>(cos->data);
    a.sin_t = static_cast<const float *>(sin->data);
    a.ld_cs = cos->row_bytes / 4;
  }
  a.k = static_cast<const float *>(k->data);
  a.ldk = ld(k);
  a.v = static_cast<const float *>(v->data);
  a.ldv = ld(v);
  a.inv_hd = inv_hd;
  a.rot = static_cast<int>(rot_dim);
  a.interleaved = interleaved != 0;
  a.heads = heads;
  a.kv_heads = kv_heads;
  return hip_status(q3::launch_seq_append(a, static_cast<hipStream_t>(stream)));
}

int page_bounds(const q3_paged_kv *kv, const q3_seqs *seqs, uint32_t rows, int kv_heads, const q3_view *bounds,
                const q3_view *bscale, void *stream) {
  q3::PageBoundsArgs a{};
  Q3_TRY(seq_common(kv, seqs, rows, kv_heads, a.pool, a.seqs));
  Q3_TRY(check_view(bounds, Q3_DT_I8));
  if (bounds->cols < 256 || bounds->rows < static_cast<uint64_t>(seqs->n_pages) * kv_heads) return Q3_ERR_VIEW;
  Q3_TRY(check_scales(bscale, seqs->n_pages, static_cast<uint32_t>(kv_heads)));
  if (bscale->col_bytes != 4) return Q3_ERR_VIEW;
  a.bounds = static_cast<int8_t *>(bounds->data);
  a.ldb = bounds->row_bytes;
  a.scale = static_cast<float *>(bscale->data);
  a.lds = bscale->row_bytes / 4;
  a.kv_heads = kv_heads;
  return hip_status(q3::launch_page_bounds(a, static_cast<hipStream_t>(stream)));
}

int varlen(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs, const q3_view *out,
           const q3_view *o8, const q3_view *os, int heads, int kv_heads, int head_dim, int causal, float qk_scale, void *ws,
           uint64_t ws_bytes, void *stream) {
  q3::SeqAttnArgs a{};
  Q3_TRY(attn_common(q8, q_scale, kv, seqs, out, o8, os, heads, kv_heads, head_dim, qk_scale, a));
  a.causal = causal != 0;
  a.ws = ws;
  Q3_TRY(check_ws(ws, ws_bytes, q3::seq_attn_ws_bytes(a)));
  return hip_status(q3::launch_seq_attn(a, static_cast<hipStream_t>(stream)));
}

int attend_pages(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs, const q3_view *ids,
                 uint32_t n_sel, const q3_view *out, const q3_view *o8, const q3_view *os, int heads, int kv_heads,
                 int head_dim, float qk_scale, void *ws, uint64_t ws_bytes, void *stream) {
  q3::SeqAttnArgs a{};
  Q3_TRY(attn_common(q8, q_scale, kv, seqs, out, o8, os, heads, kv_heads, head_dim, qk_scale, a));
  Q3_TRY(check_ids(ids, q8->rows, kv_heads, n_sel));
  if (static_cast<uint64_t>(n_sel) * kv->page_tokens > kMaxTokens) return Q3_ERR_RANGE;
  a.causal = 1;
  a.ids = static_cast<const int32_t *>(ids->data);
  a.ld_ids = ld(ids);
  a.n_sel = static_cast<int>(n_sel);
  a.ws = ws;
  Q3_TRY(check_ws(ws, ws_bytes, q3::seq_attn_ws_bytes(a)));
  return hip_status(q3::launch_seq_attn(a, static_cast<hipStream_t>(stream)));
}

int select(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs, const q3_view *bounds,
           const q3_view *bscale, const q3_view *ids, uint32_t n_sel, int heads, int kv_heads, void *ws, uint64_t ws_bytes,
           void *stream) {
  q3::SelectArgs a{};
  Q3_TRY(check_queries(q8, q_scale, heads, kv_heads));
  if (heads / kv_heads > 16) return Q3_ERR_UNSUPPORTED;
  Q3_TRY(seq_common(kv, seqs, q8->rows, kv_heads, a.pool, a.seqs));
  Q3_TRY(check_view(bounds, Q3_DT_I8));
  if (bounds->cols < 256 || bounds->rows < static_cast<uint64_t>(seqs->n_pages) * kv_heads) return Q3_ERR_VIEW;
  if (bounds->row_bytes % 16 || !aligned(bounds->data, 16)) return Q3_ERR_VIEW;
  Q3_TRY(check_scales(bscale, seqs->n_pages, static_cast<uint32_t>(kv_heads)));
  if (bscale->col_bytes != 4) return Q3_ERR_VIEW;
  Q3_TRY(check_ids(ids, q8->rows, kv_heads, n_sel));
  a.q8 = static_cast<const int8_t *>(q8->data);
  a.ldq = q8->row_bytes;
  a.qs = static_cast<const float *>(q_scale->data);
  a.ldqs = q_scale->row_bytes / 4;
  a.qs_col = q_scale->col_bytes / 4;
  a.bounds = static_cast<const int8_t *>(bounds->data);
  a.ldb = bounds->row_bytes;
  a.scale = static_cast<const float *>(bscale->data);
  a.lds = bscale->row_bytes / 4;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.n_sel = static_cast<int>(n_sel);
  a.ids = static_cast<int32_t *>(ids->data);
  a.ld_ids = ld(ids);
  a.ld_keys = score_ld(seqs, kv->page_tokens);
  a.keys = static_cast<uint32_t *>(ws);
  Q3_TRY(check_ws(ws, ws_bytes, a.ld_keys > n_sel ? 4ull * q8->rows * kv_heads * a.ld_keys : 0));
  return hip_status(q3::launch_select_pages(a, static_cast<hipStream_t>(stream)));
}

}  // namespace

extern "C" {

int q3_rope_append_paged(const q3_view *q, const q3_view *k, const q3_view *v, const q3_view *nwq, const q3_view *nwk,
                         float inv_hd, const q3_view *cos, const q3_view *sin, uint32_t rot_dim, int interleaved,
                         const q3_view *q8, const q3_view *qs, const q3_paged_kv *kv, const q3_seqs *seqs, int heads,
                         int kv_heads, void *stream) {
  return finish(append(q, k, v, nwq, nwk, inv_hd, cos, sin, rot_dim, interleaved, q8, qs, kv, seqs, heads, kv_heads, stream));
}

int q3_page_bounds(const q3_paged_kv *kv, const q3_seqs *seqs, uint32_t rows, int kv_heads, const q3_view *bounds,
                   const q3_view *bscale, void *stream) {
  return finish(page_bounds(kv, seqs, rows, kv_heads, bounds, bscale, stream));
}

int q3_attention_varlen_paged(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs,
                              const q3_view *out, const q3_view *o8, const q3_view *os, int heads, int kv_heads,
                              int head_dim, int causal, float qk_scale, void *ws, uint64_t ws_bytes, void *stream) {
  return finish(varlen(q8, q_scale, kv, seqs, out, o8, os, heads, kv_heads, head_dim, causal, qk_scale, ws, ws_bytes, stream));
}

int q3_select_pages(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs,
                    const q3_view *bounds, const q3_view *bscale, const q3_view *ids, uint32_t n_sel, int heads,
                    int kv_heads, void *ws, uint64_t ws_bytes, void *stream) {
  return finish(select(q8, q_scale, kv, seqs, bounds, bscale, ids, n_sel, heads, kv_heads, ws, ws_bytes, stream));
}

int q3_attention_pages(const q3_view *q8, const q3_view *q_scale, const q3_paged_kv *kv, const q3_seqs *seqs,
                       const q3_view *ids, uint32_t n_sel, const q3_view *out, const q3_view *o8, const q3_view *os,
                       int heads, int kv_heads, int head_dim, float qk_scale, void *ws, uint64_t ws_bytes, void *stream) {
  return finish(attend_pages(q8, q_scale, kv, seqs, ids, n_sel, out, o8, os, heads, kv_heads, head_dim, qk_scale, ws, ws_bytes, stream));
}

int q3_seqs_workspace(const q3_seqs *seqs, uint32_t rows, uint32_t page_tokens, int heads, int kv_heads, uint32_t n_sel,
                      uint64_t *bytes) {
  if (!seqs || !bytes || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > kMaxHeads || page_tokens == 0) return Q3_ERR_ARG;
  if (seqs->n_seq > kMaxSeqs || rows > kMaxRows || seqs->max_kv > kMaxTokens || seqs->max_rows > kMaxRows ||
      page_tokens > kMaxTokens || n_sel > 65536)
    return Q3_ERR_RANGE;
  q3::SeqAttnArgs a{};
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.pool.page_tokens = static_cast<int>(page_tokens);
  a.seqs.n_seq = static_cast<int>(seqs->n_seq);
  a.seqs.rows = static_cast<int>(rows);
  a.seqs.max_rows = static_cast<int>(seqs->max_rows);
  a.seqs.max_kv = static_cast<int>(seqs->max_kv);
  uint64_t need = q3::seq_attn_ws_most(a);
  if (n_sel) {
    const int32_t any = 0;
    a.ids = &any;  // only its presence counts
    a.n_sel = static_cast<int>(n_sel);
    const uint64_t pages = q3::seq_attn_ws_most(a);
    const int64_t ld_keys = score_ld(seqs, page_tokens);
    const uint64_t scores = ld_keys > 1 ? 4ull * rows * kv_heads * ld_keys : 0;
    need = need > pages ? need : pages;
    need = need > scores ? need : scores;
  }
  *bytes = need;
  return Q3_OK;
}

}  // extern "C"
