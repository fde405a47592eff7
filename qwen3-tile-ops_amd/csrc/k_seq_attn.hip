// Attention of the rows of many sequences over the paged int8 cache.
//
//   x[key] = (q . k[key]) * (qs * qk_scale) * ks[key]    q . k exact in int32
//   out    = sum_key softmax(x)[key] * vs[key] * v[key]
//
// over the keys at or before the row's position (causal), all cached keys, or
// the keys of listed pages.  Maximum, sum and products are f32.
#include "q3_seq.h"

namespace q3 {
namespace {

constexpr int HD = 128;

// One workgroup per (row, head), 256 keys a step: a thread per key for the
// scores, then a thread per (channel, half of the keys) for P V.
__global__ void __launch_bounds__(256) seq_attn_kernel(SeqAttnArgs a) {
  __shared__ float p[256], acc_s[2][HD], red[8];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int kvh = head / (a.heads / a.kv_heads);
  const int seq = seq_of_row(a.seqs, row);
  if (seq >= a.seqs.n_seq) return;
  const SeqSpan sp = seq_span(a.seqs, seq);
  if (row < sp.r0 || row >= sp.r0 + sp.n) return;
  const int pt = a.pool.page_tokens;
  const int visible = a.causal ? sp.pos(row) + 1 : sp.kv;  // <= 0: nothing
  const int64_t keys = a.ids ? static_cast<int64_t>(a.n_sel) * pt : max(visible, 0);
  const int *q = reinterpret_cast<const int *>(a.q8 + row * a.ldq + head * HD);
  const float c = a.qs[row * a.ldqs + head * a.qs_col] * a.qk_scale;
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int64_t k0 = 0; k0 < keys; k0 += 256) {
    __shared__ int64_t vat[256];
    const int64_t i = k0 + tid;
    float x = -INFINITY;
    float sv = 0.0f;
    vat[tid] = -1;
    if (i < keys) {
      int key = static_cast<int>(i);
      if (a.ids) {
        const int id = a.ids[row * a.ld_ids + kvh * a.n_sel + i / pt];
        key = id >= 0 && id <= (a.seqs.max_kv - 1) / pt ? id * pt + static_cast<int>(i % pt) : -1;
      }
      if (key >= 0 && key < visible) {
        const int page = seq_page(a.seqs, a.pool, seq, key / pt);
        if (page >= 0) {
          const int t = key % pt;
          const int *k = reinterpret_cast<const int *>(a.pool.k + page * a.pool.page_bytes + t * a.pool.row_bytes + kvh * HD);
          int dot = 0;
          for (int j = 0; j < HD / 4; ++j) dot = __builtin_amdgcn_sdot4(q[j], k[j], dot, false);
          const int64_t at = page * a.pool.spage + t * a.pool.srow + kvh;
          x = static_cast<float>(dot) * a.pool.ks[at] * c;
          sv = a.pool.vs[at];
          vat[tid] = page * a.pool.page_bytes + t * a.pool.row_bytes + kvh * HD;
        }
      }
    }
    const float w = max64(x);
    if ((tid & 63) == 0) red[tid >> 6] = w;
    __syncthreads();
    const float m1 = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float base = m1 == -INFINITY ? 0.0f : m1;
    const float e = vat[tid] >= 0 ? expf(x - base) : 0.0f;
    const float scale = expf(m - base);
    m = m1;
    p[tid] = vat[tid] >= 0 ? e * sv : 0.0f;
    float t = e;
    for (int d = 1; d < 64; d *= 2) t += __shfl_xor(t, d);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = t;
    __syncthreads();
    l = l * scale + (red[4] + red[5] + red[6] + red[7]);
    acc *= scale;
    const int ch = tid & 127, half = tid >> 7;
    for (int j = half * 128; j < half * 128 + 128; ++j)
      if (vat[j] >= 0) acc += p[j] * static_cast<float>(a.pool.v[vat[j] + ch]);
    __syncthreads();
  }
  acc_s[tid >> 7][tid & 127] = acc;
  __syncthreads();
  float o = 0.0f;
  if (tid < HD) {
    o = acc_s[0][tid] + acc_s[1][tid];
    o = l == 0.0f && m == -INFINITY ? 0.0f : o / l;
    if (a.out) a.out[row * a.ldo + head * HD + tid] = o;
  }
  if (!a.o8) return;
  const float pk = max64(fabsf(o));
  if ((tid & 63) == 0) red[tid >> 6] = pk;
  __syncthreads();
  if (tid >= HD) return;
  const float sc = __fmul_rn(fmaxf(red[0], red[1]), inv127());
  a.o8[row * a.ldo8 + head * HD + tid] = static_cast<int8_t>(quant1(o, sc));
  if (tid == 0) a.os[row * a.ldos + head * a.os_col] = sc;
}

}  // namespace

uint64_t seq_attn_ws_bytes(const SeqAttnArgs &a) { return 0; }

hipError_t launch_seq_attn(const SeqAttnArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  hipLaunchKernelGGL(seq_attn_kernel, dim3(static_cast<unsigned>(static_cast<int64_t>(a.seqs.rows) * a.heads)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace q3
