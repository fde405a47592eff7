// The pages that a row attends to, chosen by a bound of its scores.
//
// With lo, hi the int8 channel bounds of a page and KV head and b their scale,
//   score = RN(RN(f32(sum_d q_d > 0 ? q_d hi_d : q_d lo_d) * b) * qs)
// bounds q . k * qs over the page's keys from above; a KV head's score is the
// largest of its query heads'.  The sum is exact in int32, so the order of pages
// hangs on no order of summation: ties and all, it is the same everywhere.  A NaN
// score counts as the largest (its page's keys are unknown).
#include "q3_seq.h"

namespace q3 {
namespace {

constexpr int HD = 128;

// One thread per page: the ordered key of its score.
__global__ void __launch_bounds__(256) page_score_kernel(SelectArgs a) {
  const int row = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads;
  const int seq = seq_of_row(a.seqs, row);
  if (seq >= a.seqs.n_seq) return;
  const SeqSpan sp = seq_span(a.seqs, seq);
  if (row < sp.r0 || row >= sp.r0 + sp.n || sp.pos(row) < 0) return;
  const int last = sp.pos(row) / a.pool.page_tokens;
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= last || last < a.n_sel) return;
  const int page = seq_page(a.seqs, a.pool, seq, i);
  uint32_t best = 0;
  if (page >= 0) {
    const int8_t *b = a.bounds + (static_cast<int64_t>(page) * a.kv_heads + head) * a.ldb;
    const float bs = a.scale[page * a.lds + head];
    const int g = a.heads / a.kv_heads;
    for (int h = head * g; h < head * g + g; ++h) {
      const int8_t *q = a.q8 + row * a.ldq + h * HD;
      int sum = 0;
      for (int d = 0; d < HD; ++d) sum += q[d] * (q[d] > 0 ? b[HD + d] : b[d]);
      const float x = __fmul_rn(__fmul_rn(static_cast<float>(sum), bs), a.qs[row * a.ldqs + h * a.qs_col]);
      best = max(best, x != x ? 0xFFFFFFFFu : ordered_key(x));
    }
  }
  a.keys[static_cast<int64_t>(blockIdx.x) * a.ld_keys + i] = best;
}

// One workgroup per (row, KV head): the n_sel - 1 largest keys (ties to the lowest
// page) and the row's own page, in ascending order.  The threshold comes byte by
// byte from histograms of the keys that share its leading bytes; counts are
// integers, so the atomics' order changes nothing.
__global__ void __launch_bounds__(256) page_pick_kernel(SelectArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[2];
  __shared__ uint32_t tot[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads;
  const int seq = seq_of_row(a.seqs, row);
  if (seq >= a.seqs.n_seq) return;
  const SeqSpan sp = seq_span(a.seqs, seq);
  if (row < sp.r0 || row >= sp.r0 + sp.n) return;
  int32_t *ids = a.ids + row * a.ld_ids + static_cast<int64_t>(head) * a.n_sel;
  const int last = sp.pos(row) < 0 ? -1 : sp.pos(row) / a.pool.page_tokens;
  if (last < a.n_sel) {  // every page fits
    for (int i = tid; i < a.n_sel; i += 256) ids[i] = i <= last ? i : -1;
    return;
  }
  const uint32_t *keys = a.keys + static_cast<int64_t>(blockIdx.x) * a.ld_keys;
  uint32_t want = a.n_sel - 1, prefix = 0;  // keys above prefix's bytes are in
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < last; i += 256) {
      const uint32_t k = keys[i];
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t n = 0;
      int b = 255;
      while (b > 0 && n + hist[b] < want) n += hist[b--];
      found[0] = b;
      found[1] = n;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    want -= found[1];
  }
  // keys above the threshold are in, of those equal to it the first `want`
  uint32_t above = 0, equal = 0;
  if (a.n_sel > 1) {
    for (int i0 = 0; i0 < last; i0 += 256) {
      const int i = i0 + tid;
      const uint32_t k = i < last ? keys[i] : 0;
      const bool gt = i < last && k > prefix, eq = i < last && k == prefix;
      const uint64_t mg = __ballot(gt), me = __ballot(eq), under = (1ull << lane) - 1;
      if (lane == 0) tot[0][wave] = __popcll(mg), tot[1][wave] = __popcll(me);
      __syncthreads();
      uint32_t ng = above, ne = equal;
      for (int w = 0; w < wave; ++w) ng += tot[0][w], ne += tot[1][w];
      ng += __popcll(mg & under);
      ne += __popcll(me & under);
      if (gt || (eq && ne < want)) ids[ng + min(ne, want)] = i;
      for (int w = 0; w < 4; ++w) above += tot[0][w], equal += tot[1][w];
      __syncthreads();
    }
  }
  if (tid == 0) ids[a.n_sel - 1] = last;
}

}  // namespace

hipError_t launch_select_pages(const SelectArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  const unsigned items = static_cast<unsigned>(static_cast<int64_t>(a.seqs.rows) * a.kv_heads);
  const int pages = (a.seqs.max_kv + a.pool.page_tokens - 1) / a.pool.page_tokens;
  if (pages > a.n_sel) {
    hipLaunchKernelGGL(page_score_kernel, dim3(items, (pages + 255) / 256), dim3(256), 0, s, a);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(page_pick_kernel, dim3(items), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace q3
