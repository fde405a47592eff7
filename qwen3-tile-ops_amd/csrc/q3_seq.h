// The operators on the rows of many sequences over one pool of K/V pages
// (include/q3ops.h, "Batches of sequences"): kernel arguments, the lookups that
// their kernels share, and the launchers.
//
// Row starts, lengths and page tables are read on the device, so nothing on the
// host vouches for them.  Every lookup below clamps what it reads: a start or a
// length to what the host was told, a page id to the pool.  Whatever the arrays
// hold, no kernel reads or writes outside its operands.
#pragma once

#include "q3_device.h"

namespace q3 {

// The pool (q3_paged_kv without its table), strides in elements.
struct Pool {
  int8_t *k, *v;
  float *ks, *vs;
  int64_t page_bytes, row_bytes;    // of K and V rows
  int64_t spage, srow;              // of their scales, in floats
  int page_tokens, n_pages;
};

// q3_seqs with the call's row count.
struct Seqs {
  const int32_t *start, *kv_len;
  const uint16_t *tables;
  int64_t ld_table;
  int n_seq, rows, max_rows, max_kv;
};

// Whether a launch over parts of the sequences, `most` of one, names the parts one by
// one (nth_part), or has workgroups for `most` parts of every sequence: naming them takes
// a step per 64 sequences in every workgroup.  us, named / not: scores of 63 decoding
// rows and a chunk of 512 with a max_kv of 131072, 64 parts, 56 / 286; bounds of the same,
// 17 parts, 7.8 / 11.6; bounds of 2000 decoding rows and a prompt of 512 481 / 241.
inline bool name_parts(const Seqs &q, int64_t most) { return most > 1 && q.n_seq <= 32 * most; }

#if defined(__HIPCC__)

// A sequence's rows [r0, r0 + n) and its cached keys.
struct SeqSpan {
  int r0, n, kv;
  __device__ int pos(int row) const { return kv - n + (row - r0); }
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return max(lo, min(x, hi)); }

__device__ __forceinline__ SeqSpan seq_span(const Seqs &q, int begin, int end, int kv) {
  SeqSpan o;
  o.r0 = clampi(begin, 0, q.rows);
  o.n = clampi(clampi(end, 0, q.rows) - o.r0, 0, q.max_rows);
  o.kv = clampi(kv, 0, q.max_kv);
  return o;
}
__device__ __forceinline__ SeqSpan seq_span(const Seqs &q, int s) { return seq_span(q, q.start[s], q.start[s + 1], q.kv_len[s]); }

// The sequence of a row (-1: of none) and the row's position in it.
struct SeqRow {
  int seq, pos;
};

// Of the wave-uniform rows row0 .. row0 + ROWS - 1: each is in the sequence behind as
// many as end at or before it.  Of up to 64 sequences one per lane, whose starts and
// lengths come with their ends: one round trip to memory for all rows.  Of more, each
// row's 64 are found first, by the ends of 64 equal parts (starts do not decrease).
template <int ROWS>
__device__ __forceinline__ void rows_at(const Seqs &q, int row0, SeqRow (&at)[ROWS]) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = q.n_seq, begin = 0, end = INT32_MAX, kv = 0;
  auto load = [&]() {
    const int j = lane < n ? lo + lane : 0;
    begin = q.start[j], end = lane < n ? q.start[j + 1] : INT32_MAX, kv = q.kv_len[j];
  };
  if (n <= 64) load();
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    at[r] = {-1, 0};
    const int row = row0 + r;
    if (q.n_seq > 64) {
      for (lo = 0, n = q.n_seq; n > 64;) {
        const int part = (n + 63) / 64, last = min((lane + 1) * part, n) - 1;
        const int skip = min(__popcll(__ballot(q.start[lo + last + 1] <= row)) * part, n);
        lo += skip;
        n = min(part, n - skip);
      }
      load();
    }
    const int before = __popcll(__ballot(end <= row));
    if (before >= n) continue;
    const SeqSpan sp = seq_span(q, __builtin_amdgcn_readlane(begin, before), __builtin_amdgcn_readlane(end, before),
                                __builtin_amdgcn_readlane(kv, before));
    if (row >= sp.r0 && row < sp.r0 + sp.n) at[r] = {lo + before, sp.pos(row)};
  }
}
__device__ __forceinline__ SeqRow row_at(const Seqs &q, int row) {
  SeqRow at[1];
  rows_at<1>(q, row, at);
  return at[0];
}

// The sequence, and which of its parts, of the unit-th of all sequences' parts
// (parts(span) of each; seq -1 behind the last): a launch then needs no workgroups for as
// many parts of every sequence as the longest may have.
struct SeqPart {
  int seq, part;
};
template <class Parts>
__device__ __forceinline__ SeqPart nth_part(const Seqs &q, int unit, Parts parts) {
  const int lane = threadIdx.x & 63;
  for (int b = 0; b < q.n_seq; b += 64) {
    const int mine = b + lane < q.n_seq ? parts(seq_span(q, b + lane)) : 0;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    const int total = __builtin_amdgcn_readlane(upto, 63);
    if (unit < total) {
      const int at = __popcll(__ballot(upto <= unit));
      return {b + at, unit - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at))};
    }
    unit -= total;
  }
  return {-1, 0};
}

// Physical page of a sequence's logical page (0 <= logical * page_tokens <
// max_kv), -1 if the table names none of the pool's.
__device__ __forceinline__ int seq_page(const Seqs &q, const Pool &p, int s, int logical) {
  const int id = q.tables[s * q.ld_table + logical];
  return id < p.n_pages ? id : -1;
}

#endif  // __HIPCC__

// ---- new rows into the cache (k_seq_append.hip) ------------------------------
struct SeqAppendArgs {
  const float *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const float *nwq, *nwk;  // per-head norm gains (null: no norm)
  int64_t nwq_stride, nwk_stride;
  float inv_hd;
  const float *cos_t, *sin_t;  // [position][rot / 2]
  int64_t ld_cs;
  int rot, interleaved;
  int8_t *q8;
  int64_t ldq8;
  float *qs;
  int64_t ldqs, qs_col;
  int heads, kv_heads;
  Pool pool;
  Seqs seqs;
};
hipError_t launch_seq_append(const SeqAppendArgs &a, hipStream_t s);

struct PageBoundsArgs {
  int8_t *bounds;  // [page * kv_heads + head][256]: least, then largest
  int64_t ldb;
  float *scale;    // [page][head]
  int64_t lds;
  int kv_heads;
  Pool pool;
  Seqs seqs;
};
hipError_t launch_page_bounds(const PageBoundsArgs &a, hipStream_t s);

// ---- attention (k_seq_attn.hip) ----------------------------------------------
struct SeqAttnArgs {
  const int8_t *q8;
  int64_t ldq;
  const float *qs;
  int64_t ldqs, qs_col;
  int heads, kv_heads, causal;
  float qk_scale;
  const int32_t *ids;  // [row][kv_heads * n_sel] logical pages; null: all keys
  int64_t ld_ids;
  int n_sel;
  float *out;          // f32 rows, or
  int64_t ldo;
  bool out_words;      // (the launcher's: rows that 16-byte stores fit)
  int8_t *o8;          // int8 rows with one scale per head
  int64_t ldo8;
  float *os;
  int64_t ldos, os_col;
  void *ws;
  Pool pool;
  Seqs seqs;
};
uint64_t seq_attn_ws_bytes(const SeqAttnArgs &a);  // this call's
uint64_t seq_attn_ws_most(const SeqAttnArgs &a);   // any call's of at most these counts
hipError_t launch_seq_attn(const SeqAttnArgs &a, hipStream_t s);

// ---- page selection (k_seq_select.hip) ----------------------------------------
struct SelectArgs {
  const int8_t *q8;
  int64_t ldq;
  const float *qs;
  int64_t ldqs, qs_col;
  const int8_t *bounds;
  int64_t ldb;
  const float *scale;
  int64_t lds;
  int heads, kv_heads, n_sel;
  int32_t *ids;
  int64_t ld_ids;
  uint32_t *keys;  // workspace: [row * kv_heads + head][ld_keys]
  int64_t ld_keys;
  Pool pool;
  Seqs seqs;
};
hipError_t launch_select_pages(const SelectArgs &a, hipStream_t s);

}  // namespace q3
