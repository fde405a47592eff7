// New rows of many sequences into the paged cache: per-head RMSNorm, rotary
// positions, int8 quantisation, K and V written to their pages, Q to the rows
// that the attention reads; and the channel bounds of the written pages.
//
// Arithmetic: that of norm_rope_quant_heads (kernels/norm_rope_quant.h:17-111),
// one IEEE f32 operation at a time, so a row quantises to the same bits here
// and there.  The rotation turns the first rot columns of a head, paired as
// (i, i + rot / 2) or (2 i, 2 i + 1); the rest pass through.
#include "q3_seq.h"

namespace q3 {
namespace {

constexpr int HD = 128;

// A workgroup takes 8 heads (of Q, K and V in this order) of one row, 32 lanes a
// head, 4 columns a lane: a head's reads and writes are then whole 16- and 4-byte
// words, its 32-column norm blocks 8 lanes each, and a decoding row of 16 + 2 x 8
// heads is 4 workgroups.  Bound by the reads (1 KiB a wave) at many rows, by the
// chain start -> length -> page and angles -> store at one.
// VEC: x rows, gains' and angles' accesses may be 16-byte words.
template <bool VEC>
__global__ void __launch_bounds__(256) seq_append_kernel(SeqAppendArgs a, int groups) {
  __shared__ __align__(16) float ex[8][HD];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int row = blockIdx.x / groups, group = blockIdx.x % groups;
  const int slot = wave * 2 + (lane >> 5), item = group * 8 + slot;
  const int c0 = 4 * (lane & 31);
  const bool is_q = item < a.heads, is_v = item >= a.heads + a.kv_heads;
  const bool live = item < a.heads + 2 * a.kv_heads;
  const int head = is_q ? item : is_v ? item - a.heads - a.kv_heads : item - a.heads;

  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (live) {
    const float *src = (is_q   ? a.q + static_cast<int64_t>(row) * a.ldq
                        : is_v ? a.v + static_cast<int64_t>(row) * a.ldv
                               : a.k + static_cast<int64_t>(row) * a.ldk) +
                       static_cast<int64_t>(head) * HD + c0;
    if constexpr (VEC) {
      const float4 t = *reinterpret_cast<const float4 *>(src);
      x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = src[i];
    }
  }

  const int seq = seq_of_row(a.seqs, row);
  if (seq >= a.seqs.n_seq) return;  // behind the last sequence
  const SeqSpan sp = seq_span(a.seqs, seq);
  const int pos = sp.pos(row);
  if (row < sp.r0 || row >= sp.r0 + sp.n || pos < 0) return;  // uniform in the workgroup

  const float *nw = is_v ? nullptr : is_q ? a.nwq : a.nwk;
  if (a.nwq || a.nwk) {
    float s = __fadd_rn(__fadd_rn(__fmul_rn(x[0], x[0]), __fmul_rn(x[1], x[1])),
                        __fadd_rn(__fmul_rn(x[2], x[2]), __fmul_rn(x[3], x[3])));
    s = __fadd_rn(s, lane_xor<1>(s));
    s = __fadd_rn(s, lane_xor<2>(s));
    s = __fadd_rn(s, lane_xor<4>(s));
    float ss = 0.0f;
#pragma unroll
    for (int b = 0; b < 4; ++b) ss = __fadd_rn(ss, __shfl(s, (lane & 32) + 8 * b));
    if (nw && live) {
      const float rinv = rms_factor(ss, a.inv_hd);
      const int64_t ws = is_q ? a.nwq_stride : a.nwk_stride;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], rinv), nw[(c0 + i) * ws]);
    }
  }

  if (a.rot > 0) {
    const int h = a.rot / 2;
    const float *cs = a.cos_t + pos * a.ld_cs, *sn = a.sin_t + pos * a.ld_cs;
    *reinterpret_cast<float4 *>(&ex[slot][c0]) = make_float4(x[0], x[1], x[2], x[3]);
    // the 32 lanes of a head are in one wave: its own LDS writes are done
    // before its reads
    __builtin_amdgcn_wave_barrier();
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i;
        if (c < a.rot) {
          const bool first = a.interleaved ? !(c & 1) : c < h;
          const int at = a.interleaved ? c >> 1 : first ? c : c - h;
          const float o = ex[slot][a.interleaved ? c ^ 1 : first ? c + h : c - h];
          x[i] = first ? __fsub_rn(__fmul_rn(x[i], cs[at]), __fmul_rn(o, sn[at]))
                       : __fadd_rn(__fmul_rn(o, sn[at]), __fmul_rn(x[i], cs[at]));
        }
      }
    }
  }

  const float m = max32(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
  if (!live) return;
  const float scale = __fmul_rn(m, inv127());
  const double y = rcp64(scale);
  char4 q;
  q.x = static_cast<signed char>(quant_rcp(x[0], y));
  q.y = static_cast<signed char>(quant_rcp(x[1], y));
  q.z = static_cast<signed char>(quant_rcp(x[2], y));
  q.w = static_cast<signed char>(quant_rcp(x[3], y));
  int8_t *dst;
  float *sdst;
  if (is_q) {
    dst = a.q8 + static_cast<int64_t>(row) * a.ldq8;
    sdst = a.qs + static_cast<int64_t>(row) * a.ldqs + static_cast<int64_t>(head) * a.qs_col;
  } else {
    const int logical = pos / a.pool.page_tokens, t = pos % a.pool.page_tokens;
    const int page = seq_page(a.seqs, a.pool, seq, logical);
    if (page < 0) return;
    dst = (is_v ? a.pool.v : a.pool.k) + page * a.pool.page_bytes + t * a.pool.row_bytes;
    sdst = (is_v ? a.pool.vs : a.pool.ks) + page * a.pool.spage + t * a.pool.srow + head;
  }
  *reinterpret_cast<char4 *>(dst + static_cast<int64_t>(head) * HD + c0) = q;
  if ((lane & 31) == 0) *sdst = scale;
}

// Channel bounds of one page and KV head: over the page's cached keys the least
// and the largest dequantised value of each channel, rounded outwards to int8
// with one scale, so that a score computed from them is no less than any key's
// (but for the scale's own rounding).  Minima and maxima do not hang on the order,
// and the page is read anew on every call: rewritten slots leave no trace.
// One workgroup per (page, head): 8 lanes a key (16 bytes each), 32 keys a step.
// A page written by this call has just left the caches' write path, so the 4 KiB
// of a 32-token page and head come from L2.
__global__ void __launch_bounds__(256) page_bounds_kernel(PageBoundsArgs a, int pages_per_seq) {
  __shared__ float lo_s[4][HD], hi_s[4][HD];
  __shared__ float peak[2];
  const int s = blockIdx.y;
  const int head = blockIdx.x % a.kv_heads, nth = blockIdx.x / a.kv_heads;
  const SeqSpan sp = seq_span(a.seqs, s);
  const int pt = a.pool.page_tokens;
  if (sp.n == 0 || sp.kv == 0) return;
  const int logical = max(sp.kv - sp.n, 0) / pt + nth;
  if (static_cast<int64_t>(logical) * pt >= sp.kv) return;
  const int page = seq_page(a.seqs, a.pool, s, logical);
  if (page < 0) return;
  const int tokens = min(pt, sp.kv - logical * pt);
  const int tid = threadIdx.x, chunk = tid & 7;

  float lo[16], hi[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
  const int8_t *k = a.pool.k + page * a.pool.page_bytes + static_cast<int64_t>(head) * HD + 16 * chunk;
  const float *ks = a.pool.ks + page * a.pool.spage + head;
  for (int t = tid >> 3; t < tokens; t += 32) {
    const int4 w = *reinterpret_cast<const int4 *>(k + t * a.pool.row_bytes);
    const float sc = ks[t * a.pool.srow];
    const int ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = __fmul_rn(static_cast<float>(static_cast<int8_t>(ww[i >> 2] >> (8 * (i & 3)))), sc);
      lo[i] = fminf(lo[i], x);
      hi[i] = fmaxf(hi[i], x);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    lo[i] = fminf(lo[i], lane_xor<8>(lo[i]));
    lo[i] = fminf(lo[i], lane_xor<16>(lo[i]));
    lo[i] = fminf(lo[i], lane_xor<32>(lo[i]));
    hi[i] = fmaxf(hi[i], lane_xor<8>(hi[i]));
    hi[i] = fmaxf(hi[i], lane_xor<16>(hi[i]));
    hi[i] = fmaxf(hi[i], lane_xor<32>(hi[i]));
  }
  const int wave = tid >> 6;
  if ((tid & 63) < 8) {
#pragma unroll
    for (int i = 0; i < 16; ++i) lo_s[wave][16 * chunk + i] = lo[i], hi_s[wave][16 * chunk + i] = hi[i];
  }
  __syncthreads();
  float l = 0.0f, h = 0.0f;
  if (tid < HD) {
    l = fminf(fminf(lo_s[0][tid], lo_s[1][tid]), fminf(lo_s[2][tid], lo_s[3][tid]));
    h = fmaxf(fmaxf(hi_s[0][tid], hi_s[1][tid]), fmaxf(hi_s[2][tid], hi_s[3][tid]));
    const float m = max64(fmaxf(fabsf(l), fabsf(h)));
    if ((tid & 63) == 0) peak[tid >> 6] = m;
  }
  __syncthreads();
  if (tid >= HD) return;
  const float scale = __fmul_rn(fmaxf(peak[0], peak[1]), inv127());
  const double y = rcp64(scale);
  // RN32(x / scale) as in quant_rcp
  const float ql = __double2float_rn(__dmul_rn(static_cast<double>(l), y));
  const float qh = __double2float_rn(__dmul_rn(static_cast<double>(h), y));
  const float fl = (ql != ql) ? 0.0f : fminf(127.0f, fmaxf(-127.0f, floorf(ql)));
  const float fh = (qh != qh) ? 0.0f : fminf(127.0f, fmaxf(-127.0f, ceilf(qh)));
  int8_t *out = a.bounds + (static_cast<int64_t>(page) * a.kv_heads + head) * a.ldb;
  out[tid] = static_cast<int8_t>(fl);
  out[HD + tid] = static_cast<int8_t>(fh);
  if (tid == 0) a.scale[page * a.lds + head] = scale;
}

}  // namespace

hipError_t launch_seq_append(const SeqAppendArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  const int groups = (a.heads + 2 * a.kv_heads + 7) / 8;
  const auto al16 = [](const void *p, int64_t ld_) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld_ & 3) == 0; };
  const bool vec = (!a.q || al16(a.q, a.ldq)) && al16(a.k, a.ldk) && al16(a.v, a.ldv);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.seqs.rows) * groups));
  if (vec)
    hipLaunchKernelGGL(seq_append_kernel<true>, grid, dim3(256), 0, s, a, groups);
  else
    hipLaunchKernelGGL(seq_append_kernel<false>, grid, dim3(256), 0, s, a, groups);
  return hipGetLastError();
}

hipError_t launch_page_bounds(const PageBoundsArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  const int pt = a.pool.page_tokens;
  const int per = (min(a.seqs.max_rows, a.seqs.max_kv) + pt - 2) / pt + 1;  // pages that max_rows tokens can lie in
  hipLaunchKernelGGL(page_bounds_kernel, dim3(static_cast<unsigned>(per * a.kv_heads), a.seqs.n_seq), dim3(256), 0, s, a, per);
  return hipGetLastError();
}

}  // namespace q3
