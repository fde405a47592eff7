// The pages that a row attends to, chosen by a bound of its scores.
//
// With lo, hi the int8 channel bounds of a page and KV head and b their scale,
//   score = RN(RN(f32(sum_d q_d > 0 ? q_d hi_d : q_d lo_d) * b) * qs)
// bounds q . k * qs over the page's keys from above; a KV head's score is the
// largest of its query heads'.  The sum is exact in int32, so the order of pages
// hangs on no order of summation: ties and all, it is the same everywhere.  A NaN
// score counts as the largest (its page's keys are unknown).
#include "q3_attn_v.h"
#include "q3_seq.h"

namespace q3 {
namespace {

constexpr int SCORE_PAGES = 256;  // of a workgroup, 64 to a wave
constexpr int PICK_REGS = 16;     // keys that a thread of the pick holds
constexpr int PICK_MOST = 256 * PICK_REGS;

// Scores of 256 pages for up to 16 (row, query head) columns of one KV head.  With
// q's negative and positive parts side by side as the B operand, the sum is one
// [16 pages][256] x [256][16 columns] int8 product, four MFMAs; a page's 256 bytes
// are read once for the columns of all its rows.  Bound by those reads where a
// sequence has few rows: a wave has the 16 KiB of its 64 pages in flight at once,
// and the workgroups of a long context fill the CUs.  One row over 1024 pages takes 7.6
// us, 24 rows of 64 heads over 170 on average 7.7: the chain length -> table -> bounds.
__global__ void __launch_bounds__(256) page_score_kernel(SelectArgs a, int tile_rows, int tiles, bool named) {
  __shared__ __align__(16) uint32_t key_s[4][16][20];  // [column][page of a 16-page group]
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int col = lane & 15, quarter = lane >> 4;
  const int g = a.heads / a.kv_heads;
  const int head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
  const SeqPart at = !named ? SeqPart{unit / tiles, unit % tiles}
                            : nth_part(a.seqs, unit, [&](const SeqSpan &sp) { return (sp.n + tile_rows - 1) / tile_rows; });
  if (at.seq < 0) return;
  const int seq = at.seq, tile = at.part;
  const SeqSpan sp = seq_span(a.seqs, seq);
  const int row0 = sp.r0 + tile * tile_rows;
  const int rows = min(sp.r0 + sp.n - row0, tile_rows);
  if (rows <= 0) return;
  // (the tile's last row sees the most pages; its own page needs no score)
  const int most = sp.pos(row0 + rows - 1) < 0 ? 0 : sp.pos(row0 + rows - 1) / a.pool.page_tokens;
  const int page0 = blockIdx.y * SCORE_PAGES + wave * (SCORE_PAGES / 4);
  if (most < a.n_sel || page0 >= most) return;

  // bounds of 64 pages, one table entry a lane
  const int mine = page0 + lane < most ? seq_page(a.seqs, a.pool, seq, page0 + lane) : -1;
  v4i_d bf[4][4];
  float bs[4][4];
  bool in[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int page = __shfl(mine, 16 * t + col);
    const int8_t *b = a.bounds + (static_cast<int64_t>(max(page, 0)) * a.kv_heads + head) * a.ldb + 16 * quarter;
#pragma unroll
    for (int i = 0; i < 4; ++i) bf[t][i] = page < 0 ? v4i_d{0, 0, 0, 0} : *reinterpret_cast<const v4i_d *>(b + 64 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // of the pages that this lane's results are for
      const int p = __shfl(mine, 16 * t + 4 * quarter + i);
      in[t][i] = p >= 0;
      bs[t][i] = p >= 0 ? a.scale[p * a.lds + head] : 0.0f;
    }
  }

  // q as the B operand: column (row, query head), 16 bytes of each 64
  const int r = col / g, h = head * g + col % g;
  const bool live = r < rows;
  v4i_d qf[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
  float qs = 0.0f;
  if (live) {
    const int8_t *q = a.q8 + (row0 + r) * a.ldq + h * HD + 16 * quarter;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const v4i_d w = *reinterpret_cast<const v4i_d *>(q + 64 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t neg = ((static_cast<uint32_t>(w[j]) >> 7) & 0x01010101u) * 255u;  // 255 in the bytes below 0
        qf[i][j] = static_cast<int>(w[j] & neg);
        qf[2 + i][j] = static_cast<int>(w[j] & ~neg);
      }
    }
    qs = a.qs[(row0 + r) * a.ldqs + h * a.qs_col];
  }

#pragma unroll
  for (int t = 0; t < 4; ++t) {
    v4i_d s = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[t][i], qf[i], s, 0, 0, 0);
    uint32_t k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = __fmul_rn(__fmul_rn(static_cast<float>(s[i]), bs[t][i]), qs);
      k[i] = !in[t][i] ? 0u : x != x ? 0xFFFFFFFFu : ordered_key(x);
    }
    // the largest of a row's query heads: its wave's own 16 x 16 keys through LDS
    *reinterpret_cast<uint4 *>(&key_s[wave][col][4 * quarter]) = make_uint4(k[0], k[1], k[2], k[3]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int page = page0 + 16 * t + col;
    for (int rr = quarter; rr < rows; rr += 4) {
      uint32_t best = 0;
      for (int j = 0; j < g; ++j) best = max(best, key_s[wave][rr * g + j][col]);
      if (page < most) a.keys[(static_cast<int64_t>(row0 + rr) * a.kv_heads + head) * a.ld_keys + page] = best;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// One workgroup per (row, KV head): the n_sel - 1 largest keys (ties to the lowest
// page) and the row's own page, in ascending order.  The threshold is the largest
// value that enough keys reach, found two bits a round by counting, until exactly as
// many reach it as are wanted; wave w has the w-th quarter of the pages, so a page's
// place needs the waves' totals alone.
// REGS: the keys stay in registers (4096 pages); otherwise each round reads them.
// 64 of 1024 pages take 7.7 us (all 16 rounds 9.0), 33 of 170 for 192 (row, head) pairs
// 6.4: the chain length -> keys -> rounds, each a barrier.
template <bool REGS>
__global__ void __launch_bounds__(256) page_pick_kernel(SelectArgs a) {
  __shared__ uint32_t count_s[2][3][4];
  __shared__ uint32_t total_s[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int row = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads;
  const SeqRow at = row_at(a.seqs, row);
  if (at.seq < 0) return;
  int32_t *ids = a.ids + row * a.ld_ids + static_cast<int64_t>(head) * a.n_sel;
  const int last = at.pos < 0 ? -1 : at.pos / a.pool.page_tokens;
  if (last < a.n_sel) {  // every page fits
    for (int i = tid; i < a.n_sel; i += 256) ids[i] = i <= last ? i : -1;
    return;
  }
  const uint32_t want = a.n_sel - 1;
  if (want == 0) {
    if (tid == 0) ids[0] = last;
    return;
  }
  const uint32_t *keys = a.keys + static_cast<int64_t>(blockIdx.x) * a.ld_keys;
  // key j of lane l in wave w is page base + 64 j + l
  const int each = (last + 255) / 256;
  const int base = wave * each * 64 + lane;
  uint32_t reg[REGS ? PICK_REGS : 1];
  if constexpr (REGS) {
#pragma unroll
    for (int j = 0; j < PICK_REGS; ++j) {
      const int i = base + 64 * j;
      reg[j] = j < each && i < last ? keys[i] : 0;
    }
  }
  // f(key, page) over the wave's pages; a lane behind the last has key 0 and page -1
  auto each_key = [&](auto f) {
    if constexpr (REGS) {
#pragma unroll
      for (int j = 0; j < PICK_REGS; ++j)
        if (j < each) f(reg[j], base + 64 * j < last ? base + 64 * j : -1);
    } else {
      for (int j = 0; j < each; ++j) {
        const int i = base + 64 * j;
        f(i < last ? keys[i] : 0u, i < last ? i : -1);
      }
    }
  };
  uint32_t prefix = 0;
  for (int round = 0; round < 16; ++round) {
    const int shift = 30 - 2 * round;
    const uint32_t t1 = prefix | (1u << shift), t2 = prefix | (2u << shift), t3 = prefix | (3u << shift);
    uint32_t c1 = 0, c2 = 0, c3 = 0;  // (a lane behind the last is below every threshold)
    each_key([&](uint32_t k, int) {
      c1 += __popcll(__ballot(k >= t1));
      c2 += __popcll(__ballot(k >= t2));
      c3 += __popcll(__ballot(k >= t3));
    });
    uint32_t(&count)[3][4] = count_s[round & 1];
    if (lane == 0) count[0][wave] = c1, count[1][wave] = c2, count[2][wave] = c3;
    __syncthreads();
    c1 = c2 = c3 = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) c1 += count[0][w], c2 += count[1][w], c3 += count[2][w];
    const uint32_t reach = c3 >= want ? c3 : c2 >= want ? c2 : c1;
    prefix = c3 >= want ? t3 : c2 >= want ? t2 : c1 >= want ? t1 : prefix;
    if (reach == want) break;  // no key between: the bits below do not matter
  }
  // keys above the threshold are in, of those equal to it the first ones
  uint32_t above = 0, equal = 0;
  each_key([&](uint32_t k, int i) {
    above += __popcll(__ballot(i >= 0 && k > prefix));
    equal += __popcll(__ballot(i >= 0 && k == prefix));
  });
  if (lane == 0) total_s[0][wave] = above, total_s[1][wave] = equal;
  __syncthreads();
  uint32_t ng = 0, ne = 0, all = 0;  // before this wave, and those above in all
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) ng += total_s[0][w], ne += total_s[1][w];
    all += total_s[0][w];
  }
  const uint32_t need = want - all;
  const uint64_t under = (1ull << lane) - 1;
  each_key([&](uint32_t k, int i) {
    const bool gt = i >= 0 && k > prefix, eq = i >= 0 && k == prefix;
    const uint64_t mg = __ballot(gt), me = __ballot(eq);
    const uint32_t g = ng + __popcll(mg & under), e = ne + __popcll(me & under);
    if (gt || (eq && e < need)) ids[g + min(e, need)] = i;
    ng += __popcll(mg);
    ne += __popcll(me);
  });
  if (tid == 0) ids[want] = last;
}

}  // namespace

hipError_t launch_select_pages(const SelectArgs &a, hipStream_t s) {
  if (a.seqs.rows == 0 || a.seqs.n_seq == 0) return hipSuccess;
  const int64_t items = static_cast<int64_t>(a.seqs.rows) * a.kv_heads;
  const int pages = (a.seqs.max_kv + a.pool.page_tokens - 1) / a.pool.page_tokens;
  if (pages > a.n_sel) {
    const int tile_rows = 16 * a.kv_heads / a.heads;
    const int tiles = (max(a.seqs.max_rows, 1) + tile_rows - 1) / tile_rows;
    // (row tiles of all sequences: at most)
    const int64_t each = static_cast<int64_t>(a.seqs.n_seq) * tiles, all = a.seqs.rows / tile_rows + a.seqs.n_seq;
    const bool named = name_parts(a.seqs, tiles) && all < each;
    const int64_t units = (named ? all : each) * a.kv_heads;
    const int64_t chunks = (pages + SCORE_PAGES - 1) / SCORE_PAGES;
    if (units > INT32_MAX / 256 || chunks > 65535 || units * chunks > INT32_MAX / 256) return hipErrorInvalidValue;
    hipLaunchKernelGGL(page_score_kernel, dim3(static_cast<unsigned>(units), static_cast<unsigned>(chunks)), dim3(256), 0, s, a,
                       tile_rows, tiles, named);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (items > INT32_MAX / 256) return hipErrorInvalidValue;
  if (pages <= PICK_MOST)
    hipLaunchKernelGGL(page_pick_kernel<true>, dim3(static_cast<unsigned>(items)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(page_pick_kernel<false>, dim3(static_cast<unsigned>(items)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace q3
