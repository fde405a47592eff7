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
constexpr int64_t APPEND_WGS = 1024;

// Four values as int8 with their head's scale: quant_rcp's results, with its f64
// arithmetic (half of this kernel's time) only where a quotient lies near a half.
// x * rcp(scale) is within 127 * 3 * 2^-24 < 3e-5 of x / scale where the scale is a
// normal number whose reciprocal is one too, so elsewhere both round alike.
__device__ __forceinline__ char4 quant4(const float (&x)[4], float scale) {
  const float inv = __builtin_amdgcn_rcpf(scale);
  float r[4];
  bool sure = scale > 0x1p-100f && scale < 0x1p+100f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = __fmul_rn(x[i], inv);
    r[i] = rintf(t);
    sure &= fabsf(__fsub_rn(t, r[i])) < 0.4999f;
    r[i] = fminf(127.0f, fmaxf(-127.0f, r[i]));
  }
  char4 q;
  q.x = static_cast<signed char>(r[0]);
  q.y = static_cast<signed char>(r[1]);
  q.z = static_cast<signed char>(r[2]);
  q.w = static_cast<signed char>(r[3]);
  if (__ballot(!sure)) {
    const double y = rcp64(scale);
    q.x = static_cast<signed char>(quant_rcp(x[0], y));
    q.y = static_cast<signed char>(quant_rcp(x[1], y));
    q.z = static_cast<signed char>(quant_rcp(x[2], y));
    q.w = static_cast<signed char>(quant_rcp(x[3], y));
  }
  return q;
}

// ((b0 + b1) + b2) + b3 of the four 8-lane groups' sums in each 32-lane half.
__device__ __forceinline__ float ordered_sum4(float s, int lane) {
  const float b = lane_xor<8>(s), c = lane_xor<16>(s);
  const float d = lane_xor<8>(c);
  const bool odd = lane & 8, second = lane & 16;
  const float lo = __fadd_rn(second ? c : s, second ? d : b);
  const float b2 = second ? (odd ? b : s) : (odd ? d : c), b3 = second ? (odd ? s : b) : (odd ? c : d);
  return __fadd_rn(__fadd_rn(lo, b2), b3);
}

// A workgroup takes 8 heads (of Q, K and V in this order) of ROWS rows, 32 lanes a
// head, 4 columns a lane: a head's reads and writes are then whole 16- and 4-byte
// words, its 32-column norm blocks 8 lanes each, and a decoding row of 16 + 2 x 8
// heads is 4 workgroups.  At one row bound by the chain start -> length -> page and
// angles -> store (4.1 us), at many by the same chain of each workgroup beside what is
// in flight: 2048 rows (43 MB) take 20.9 us, 24.3 with one row a workgroup, 22.3 with four
// (more registers, fewer waves); with no arithmetic at all it is 19.
// VEC: x rows may be read as 16-byte words; angles: so may a lane's angles (and its
// four columns are rotated alike).
template <bool VEC, int ROWS>
__global__ void __launch_bounds__(256, 8) seq_append_kernel(SeqAppendArgs a, bool angles) {
  __shared__ __align__(16) float ex[8][HD];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int row_blocks = (a.seqs.rows + ROWS - 1) / ROWS;
  const int row0 = blockIdx.x % row_blocks * ROWS, group = blockIdx.x / row_blocks;
  const int slot = wave * 2 + (lane >> 5), item = group * 8 + slot;
  const int c0 = 4 * (lane & 31);
  const bool is_q = item < a.heads, is_v = item >= a.heads + a.kv_heads;
  const bool live = item < a.heads + 2 * a.kv_heads;
  const int head = is_q ? item : is_v ? item - a.heads - a.kv_heads : item - a.heads;

  float x[ROWS][4];
  const float *src = (is_q ? a.q : is_v ? a.v : a.k) + static_cast<int64_t>(head) * HD + c0;
  const int64_t ldx = is_q ? a.ldq : is_v ? a.ldv : a.ldk;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = min(row0 + r, a.seqs.rows - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[r][i] = 0.0f;
    if (live) {
      if constexpr (VEC) {
        const float4 t = *reinterpret_cast<const float4 *>(src + row * ldx);
        x[r][0] = t.x, x[r][1] = t.y, x[r][2] = t.z, x[r][3] = t.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[r][i] = src[row * ldx + i];
      }
    }
  }

  SeqRow at[ROWS];
  rows_at<ROWS>(a.seqs, row0, at);
  int page[ROWS], slot_of[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    page[r] = -1, slot_of[r] = 0;
    if (row0 + r >= a.seqs.rows || at[r].seq < 0) at[r].pos = -1;  // of no sequence: left as it is
    if (at[r].pos < 0) continue;
    slot_of[r] = at[r].pos % a.pool.page_tokens;
    page[r] = seq_page(a.seqs, a.pool, at[r].seq, at[r].pos / a.pool.page_tokens);
  }

  float w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  const float *nw = is_v || !live ? nullptr : is_q ? a.nwq : a.nwk;
  if (nw) {
    const int64_t ws = is_q ? a.nwq_stride : a.nwk_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = nw[(c0 + i) * ws];
  }
  const int h = a.rot / 2;
  const bool first = c0 < h, turns = !is_v && live && c0 < a.rot;
  float cs[ROWS][4], sn[ROWS][4];
  if (angles) {  // (rot is a multiple of 8)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (!turns || at[r].pos < 0) continue;
      const float *c = a.cos_t + at[r].pos * a.ld_cs, *s = a.sin_t + at[r].pos * a.ld_cs;
      if (a.interleaved) {
        const float2 u = *reinterpret_cast<const float2 *>(c + (c0 >> 1)), v = *reinterpret_cast<const float2 *>(s + (c0 >> 1));
        cs[r][0] = cs[r][1] = u.x, cs[r][2] = cs[r][3] = u.y;
        sn[r][0] = sn[r][1] = v.x, sn[r][2] = sn[r][3] = v.y;
      } else {
        const float4 u = *reinterpret_cast<const float4 *>(c + (first ? c0 : c0 - h));
        const float4 v = *reinterpret_cast<const float4 *>(s + (first ? c0 : c0 - h));
        cs[r][0] = u.x, cs[r][1] = u.y, cs[r][2] = u.z, cs[r][3] = u.w;
        sn[r][0] = v.x, sn[r][1] = v.y, sn[r][2] = v.z, sn[r][3] = v.w;
      }
    }
  }

#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (at[r].pos < 0) continue;  // uniform in the workgroup
    const int row = row0 + r;
    float (&y)[4] = x[r];
    if (a.nwq || a.nwk) {
      float s = __fadd_rn(__fadd_rn(__fmul_rn(y[0], y[0]), __fmul_rn(y[1], y[1])),
                          __fadd_rn(__fmul_rn(y[2], y[2]), __fmul_rn(y[3], y[3])));
      s = __fadd_rn(s, lane_xor<1>(s));
      s = __fadd_rn(s, lane_xor<2>(s));
      s = __fadd_rn(s, lane_xor<4>(s));
      const float ss = ordered_sum4(s, lane);
      if (nw) {
        const float rinv = rms_factor(ss, a.inv_hd);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __fmul_rn(__fmul_rn(y[i], rinv), w[i]);
      }
    }
    if (a.rot > 0) {
      // (a head's 32 lanes are in one wave, which finishes its LDS writes before its
      // reads, and those before the next row's writes)
      *reinterpret_cast<float4 *>(&ex[slot][c0]) = make_float4(y[0], y[1], y[2], y[3]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (turns && angles) {
        float o[4] = {y[1], y[0], y[3], y[2]};
        if (!a.interleaved) {
          const float4 t = *reinterpret_cast<const float4 *>(&ex[slot][first ? c0 + h : c0 - h]);
          o[0] = t.x, o[1] = t.y, o[2] = t.z, o[3] = t.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool f = a.interleaved ? !(i & 1) : first;
          const float u = __fmul_rn(y[i], cs[r][i]), v = __fmul_rn(o[i], sn[r][i]);
          y[i] = f ? __fsub_rn(u, v) : __fadd_rn(v, u);
        }
      } else if (turns) {
        const float *c = a.cos_t + at[r].pos * a.ld_cs, *s = a.sin_t + at[r].pos * a.ld_cs;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = c0 + i;
          if (col < a.rot) {
            const bool f = a.interleaved ? !(col & 1) : col < h;
            const int at = a.interleaved ? col >> 1 : f ? col : col - h;
            const float o = ex[slot][a.interleaved ? col ^ 1 : f ? col + h : col - h];
            const float u = __fmul_rn(y[i], c[at]), v = __fmul_rn(o, s[at]);
            y[i] = f ? __fsub_rn(u, v) : __fadd_rn(v, u);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    const float m = max32(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
    if (!live) continue;
    const float scale = __fmul_rn(m, inv127());
    const char4 q = quant4(y, scale);
    int8_t *dst;
    float *sdst;
    if (is_q) {
      dst = a.q8 + row * a.ldq8;
      sdst = a.qs + row * a.ldqs + head * a.qs_col;
    } else {
      if (page[r] < 0) continue;
      dst = (is_v ? a.pool.v : a.pool.k) + page[r] * a.pool.page_bytes + slot_of[r] * a.pool.row_bytes;
      sdst = (is_v ? a.pool.vs : a.pool.ks) + page[r] * a.pool.spage + slot_of[r] * a.pool.srow + head;
    }
    *reinterpret_cast<char4 *>(dst + static_cast<int64_t>(head) * HD + c0) = q;
    if ((lane & 31) == 0) *sdst = scale;
  }
}

// Channel bounds of one page and KV head: over the page's cached keys the least
// and the largest dequantised value of each channel, rounded outwards to int8
// with one scale, so that a score computed from them is no less than any key's
// (but for the scale's own rounding).  Minima and maxima do not hang on the order,
// and the page is read anew on every call: rewritten slots leave no trace.
// One workgroup per (page, head): 8 lanes a key (16 bytes each), 32 keys a step.
// A page written by this call has just left the caches' write path, so the 4 KiB
// of a 32-token page and head come from L2.  781 rows of 7 sequences, 8 heads: 5.9 us, the
// chain length -> table -> keys and two barriers.
__global__ void __launch_bounds__(256) page_bounds_kernel(PageBoundsArgs a, int per, bool named) {
  __shared__ float lo_s[4][HD], hi_s[4][HD];
  __shared__ float peak[2];
  const int head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
  const int pt = a.pool.page_tokens;
  const SeqPart at = !named ? SeqPart{unit / per, unit % per} : nth_part(a.seqs, unit, [&](const SeqSpan &sp) {
    return sp.n == 0 || sp.kv == 0 ? 0 : (sp.kv - 1) / pt - max(sp.kv - sp.n, 0) / pt + 1;
  });
  if (at.seq < 0) return;
  const int s = at.seq, nth = at.part;
  const SeqSpan sp = seq_span(a.seqs, s);
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
  const bool angles = a.rot > 0 && a.rot % 8 == 0 && al16(a.cos_t, a.ld_cs) && al16(a.sin_t, a.ld_cs);
  // two rows a workgroup once one a workgroup would leave some waiting for a CU
  const bool two = vec && static_cast<int64_t>(a.seqs.rows) * groups > APPEND_WGS;
  const int64_t wgs = (two ? (a.seqs.rows + 1) / 2 : a.seqs.rows) * static_cast<int64_t>(groups);
  if (wgs > INT32_MAX / 256) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(wgs));
  if (two)
    hipLaunchKernelGGL((seq_append_kernel<true, 2>), grid, dim3(256), 0, s, a, angles);
  else if (vec)
    hipLaunchKernelGGL((seq_append_kernel<true, 1>), grid, dim3(256), 0, s, a, angles);
  else
    hipLaunchKernelGGL((seq_append_kernel<false, 1>), grid, dim3(256), 0, s, a, angles);
  return hipGetLastError();
}

hipError_t launch_page_bounds(const PageBoundsArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  const int pt = a.pool.page_tokens;
  const int64_t most = min(a.seqs.max_rows, a.seqs.max_kv), n_seq = a.seqs.n_seq;
  const int64_t per = (most + pt - 2) / pt + 1;  // pages that max_rows tokens can lie in
  // (of all rows: n lie in n / pt pages and two more at most)
  const int64_t all = a.seqs.rows / pt + 2 * n_seq;
  const bool named = name_parts(a.seqs, per) && all < n_seq * per;
  const int64_t pages = named ? all : n_seq * per;
  if (pages * a.kv_heads > INT32_MAX / 256) return hipErrorInvalidValue;
  hipLaunchKernelGGL(page_bounds_kernel, dim3(static_cast<unsigned>(pages * a.kv_heads)), dim3(256), 0, s, a,
                     static_cast<int>(per), named);
  return hipGetLastError();
}

}  // namespace q3
