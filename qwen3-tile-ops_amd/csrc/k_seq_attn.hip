// Attention of the rows of many sequences over the paged int8 cache.
//
//   x[key] = (q . k[key]) * ks[key] * (qs * qk_scale)     q . k exact in int32
//   out    = sum_key softmax(x)[key] * vs[key] * v[key]
//
// over the keys at or before the row's position (causal), all cached keys, or
// the keys of listed pages.  One pass with the running maximum and sum of the
// softmax, both in f32 and in base 2 (log2 e goes into the query's scale).
//
// The query heads of a KV head and the rows of a sequence are columns alike:
// column c is row c / group, head c % group, and K and V are read once for all
// columns of a tile.  Scores come transposed, S^T = K Q^T, so that a lane of the
// int8 MFMA's result holds keys of one column: the maximum and the sum of a column
// are register operations and two lane exchanges, and its P is already the B
// operand of O^T = V^T P^T, the keys of a step in the order in which the
// transposing LDS read delivers V.
//
// P is not rounded to 8 bits, nor to one bf16: p * vs goes to the matrix cores as
// the sum of three bf16 numbers, all of its f32 bits (measured against float64,
// 2-norm: two numbers leave 2.3e-6, three 2e-7 at 2000 keys, where f32 sums in torch leave 6e-7;
// one would leave 1.6e-3), V as bf16, which holds every int8.  bf16 because the
// range of the V scales is the user's, which f16 does not hold.
#include <algorithm>
#include <type_traits>

#include "q3_attn_v.h"
#include "q3_seq.h"

namespace q3 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;

// ---- exchanges and conversions -------------------------------------------------

// max / sum over the four 16-lane rows that share a column
__device__ __forceinline__ float col_max(float x) {
  LanePair p = lane_pair16(__float_as_uint(x));
  x = fmaxf(__uint_as_float(p.a), __uint_as_float(p.b));
  p = lane_pair32(__float_as_uint(x));
  return fmaxf(__uint_as_float(p.a), __uint_as_float(p.b));
}
__device__ __forceinline__ float col_sum(float x) {
  LanePair p = lane_pair16(__float_as_uint(x));
  x = __uint_as_float(p.a) + __uint_as_float(p.b);
  p = lane_pair32(__float_as_uint(x));
  return __uint_as_float(p.a) + __uint_as_float(p.b);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const v2f t = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(t, v2bf));
}

// x[0..7] as the sum of three bf16 numbers, the B operands of as many products
struct Bf16x3 {
  v8bf part[3];
};
__device__ __forceinline__ Bf16x3 split_bf16(const float (&x)[8]) {
  v4u w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      w[t][i] = pack_bf16(a, b);
      a -= __uint_as_float(w[t][i] << 16);
      b -= __uint_as_float(w[t][i] & 0xffff0000u);
    }
  }
  Bf16x3 r;
#pragma unroll
  for (int t = 0; t < 3; ++t) r.part[t] = __builtin_bit_cast(v8bf, w[t]);
  return r;
}

// 8 int8 as bf16, exactly
__device__ __forceinline__ v8bf int8_bf16(v2i_d w) {
  v4u r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j)));
    r[2 * i] = pack_bf16(f[0], f[1]);
    r[2 * i + 1] = pack_bf16(f[2], f[3]);
  }
  return __builtin_bit_cast(v8bf, r);
}

// The same in f16: x as two numbers (2^-22 of it while it is above 2^-3; below,
// 2^-25), int8 exactly: 0x64 over the byte with its sign bit turned is 1024 + 128 + b.
struct F16x2 {
  v8h part[2];
};
__device__ __forceinline__ F16x2 split_f16(const float (&x)[8]) {
  v4u w[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const v2f t = {x[2 * i], x[2 * i + 1]};
    w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, v2h));
    // what is left, x - h with h read as f16 (exact)
    v2f r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r.x) : "v"(w[0][i]), "v"(t.x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r.y) : "v"(w[0][i]), "v"(t.y));
    w[1][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2h));
  }
  F16x2 p;
  p.part[0] = __builtin_bit_cast(v8h, w[0]);
  p.part[1] = __builtin_bit_cast(v8h, w[1]);
  return p;
}
__device__ __forceinline__ v8h int8_f16(v2i_d w) {
  v4u r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = static_cast<uint32_t>(w[i]) ^ 0x80808080u;
    r[2 * i] = __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u);
    r[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u);
  }
  return __builtin_bit_cast(v8h, r) - static_cast<_Float16>(1152.0f);
}

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 4 bytes per lane global -> LDS (lane l writes lds + 4 l), see lds_copy16
__device__ __forceinline__ void lds_copy4(const void *src, const void *lds) {
  const uint32_t m0v =
      __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to_lds(lds))));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(m0v) : "memory", "m0");
}

// ---- the result ---------------------------------------------------------------

// 8 channels of a finished row: f32, or int8 with the head's scale, whose
// maximum is taken over the 16 lanes that hold the head's other channels.
__device__ __forceinline__ void store_row8(const SeqAttnArgs &a, int row, int head, int d0, const float (&o)[8]) {
  if (a.out) {
    float *dst = a.out + row * a.ldo + head * HD + d0;
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = o[i];
    return;
  }
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(o[i]));
  m = fmaxf(m, lane_xor<1>(m));
  m = fmaxf(m, lane_xor<2>(m));
  m = fmaxf(m, lane_xor<4>(m));
  m = fmaxf(m, lane_xor<8>(m));
  const float scale = __fmul_rn(m, inv127());
  const double y = rcp64(scale);
  int8_t *dst = a.o8 + row * a.ldo8 + head * HD + d0;
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[i] = static_cast<int8_t>(quant_rcp(o[i], y));
  if (d0 == 0) a.os[row * a.ldos + head * a.os_col] = scale;
}

// Partial results of a kernel's (row, head) slots by split: the unnormalised O,
// its maximum and its sum.
struct Partials {
  float *o;    // [slot][split][128]
  float2 *ml;  // [slot][split]
  int64_t slots;
  int splits, span;  // of a list's keys; a sequence's: split_span
};

// The keys of each of at most `splits` parts of a sequence: its length is known on the
// device alone, and max_kv may be far above it.
__device__ __forceinline__ int split_span(int keys, int splits, int least, int step) {
  return max(least, ((keys + splits - 1) / splits + step - 1) / step * step);
}

__device__ __forceinline__ float exp2_from(float x, float base) { return __builtin_amdgcn_exp2f(x - base); }

// ---- few columns: 16 to a tile -------------------------------------------------
//
// A workgroup takes one tile of 16 columns, one KV head and one split of the keys;
// its four waves take 32-key blocks in turn, each with its own running maximum and
// sum, and join at the end.  A block is K [32][128] and V [32][128] int8 and their
// 64 scales, 8.25 KiB, copied straight into the wave's own LDS, so no wave waits for
// another and what is in flight costs no registers: K into its one place once the block's
// scores are formed, V and the scales beside those of the block before.  12.5 KiB a
// wave then, and three workgroups a CU (with two places for K two: 92 rows' lists of
// pages 58 us instead of 49, 256 rows at 1000 keys 110 instead of 101; K straight to
// registers, four a CU, reads half lines: 32 rows at 16000 keys 233 us instead of 208).  16-byte chunk
// c of key r lies at chunk c ^ (r & 7) (V: c ^ vswz(r)), so that neither the K
// operand's reads (16 keys, one chunk) nor the transposing reads of V (8 keys, one
// chunk) meet in a bank.  Bound by the K/V stream once there are keys enough: one row at
// 131072 keys 56 us (4.9 TB/s), 32 rows at 16000, eight heads a KV head, 208 with the join
// (5.2); one row at 543 keys 6.7, a launch and the chain length -> table -> keys.
constexpr int KB = 32;
constexpr int FEW_COLS = 16;
constexpr int FEW_WAVES = 4;
constexpr int FEW_STAGES = 2;  // of V and the scales
constexpr int FEW_V = 0, FEW_S = KB * HD, FEW_STAGE = KB * HD + 2 * KB * 4;
constexpr int FEW_K = FEW_STAGES * FEW_STAGE, FEW_WAVE = FEW_K + KB * HD;  // bytes of a wave
constexpr int FEW_ROW = HD + 4;  // floats of a column's row where the waves join
constexpr int FEW_BLOCKS = 64 * FEW_WAVES;  // named at a time, one by a lane of each wave
// Keys of a split: a multiple of FEW_STEP, FEW_LEAST at least.  us with 128, 256, 512 and 1024
// at least, with the join: one row at 543 keys 9.6, 10.8, 12.5, 10.2, at 2000 9.8, 11.0, 12.6, 17.3, at
// 8000 13.7, 12.3, 13.5, 17.6; 24 sequences of 3 rows behind 1000 keys 23, 18, 20, 16; 64 rows
// at 500 .. 4000 keys 66.8, 66.8, 67.0, 68.5, at 300 20, 18, 13, 12.
constexpr int FEW_STEP = KB * FEW_WAVES, FEW_LEAST = 256;
static_assert(FEW_WAVES * FEW_COLS * FEW_ROW * 4 <= FEW_WAVES * FEW_WAVE, "the join fits the stages");

struct FewPlan {
  Partials part;  // slots: (sequence, KV head, column), of listed pages (row, head)
  int64_t units;  // (sequence or row) x tiles of 16 columns
  int tiles;
  int most;       // columns of a sequence that are taken here
  int each;       // workgroups of a sequence and KV head to aim at
  int by_row;     // slots lie by (row, head) in memory: fewer, where row counts are far from equal
};

// The keys of a split of a sequence, whose tiles share its part of the workgroups (so a
// decoding row beside short chunks is split as finely as among its like).  The part is the
// same for every sequence: one row at 131072 keys among 63 at 500 gets 3 splits a KV head,
// of 64 launched for it alone, and takes 713 us instead of 60.
__device__ __forceinline__ int few_span(const FewPlan &p, int keys, int cols) {
  const int tiles = (cols + FEW_COLS - 1) / FEW_COLS;
  return split_span(keys, clampi(p.each / max(tiles, 1), 1, p.part.splits), FEW_LEAST, FEW_STEP);
}

struct FewLds {
  __align__(16) uint8_t stage[FEW_WAVES * FEW_WAVE];
  float m[FEW_WAVES][FEW_COLS], l[FEW_WAVES][FEW_COLS];
};

// (block: of the workgroups that the plan asks for.)  ONCE: no other workgroup reads
// these keys, so they are read past the caches (one row at 131072 keys 69 -> 62 us, 32
// rows at 16000 232 -> 208; where rows share pages that costs: 92 rows' lists 48 -> 58).
template <bool LIST, bool ONCE>
__device__ void few_columns(const SeqAttnArgs &a, const FewPlan &p, int block, FewLds &lds) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int col = lane & 15, quarter = lane >> 4;

  // Workgroups go round the 8 XCDs.  Keys read once: the KV heads of one (unit, split)
  // share an XCD, whose L2 then holds the lines of scales that they share.  Others: a KV
  // head keeps to its XCD, whose L2 then holds the pages that rows share (92 rows' lists
  // 59 -> 48 us; 64 lists of one row each 83 -> 95).
  const int group_heads = a.heads / a.kv_heads;
  const int rest = block >> 3;
  const int kvh = ONCE ? rest % a.kv_heads : block % a.kv_heads;
  const int us = ONCE ? (rest / a.kv_heads) * 8 + (block & 7) : block / a.kv_heads;
  // Split by split: the dispatcher goes round the CUs' groups strictly, so a pattern
  // of splits with work and without would leave some of them idle.
  const int unit = us % static_cast<int>(p.units), split = us / static_cast<int>(p.units);
  if (split >= p.part.splits) return;
  const int tile = unit % p.tiles;

  const int pt = a.pool.page_tokens;

  // this lane's column, and how many keys it sees
  const int c = tile * FEW_COLS + col;
  int seq, row0, row, g, cols, sees, span = p.part.span;
  bool whole = p.part.splits == 1;
  if constexpr (LIST) {
    row0 = row = unit / p.tiles, g = c, cols = group_heads;
    const SeqRow at = row_at(a.seqs, row);
    if (at.seq < 0) return;
    seq = at.seq;
    sees = max(at.pos + 1, 0);
  } else {
    seq = unit / p.tiles;
    const SeqSpan sp = seq_span(a.seqs, seq);
    cols = sp.n * group_heads;
    if (cols > p.most || tile * FEW_COLS >= cols) return;
    span = few_span(p, sp.kv, cols);
    whole = sp.kv <= span;
    row0 = sp.r0, row = sp.r0 + c / group_heads, g = c % group_heads;
    sees = a.causal ? max(sp.pos(row) + 1, 0) : sp.kv;
  }
  const bool live = c < cols;
  if (!live) sees = 0;
  // the tile's first column sees the fewest keys, its last the most
  const int vmin = __builtin_amdgcn_readlane(sees, 0);
  const int vmax = __builtin_amdgcn_readlane(sees, min(cols - tile * FEW_COLS, FEW_COLS) - 1);

  const int span_blocks = span / KB;
  if constexpr (!LIST) {  // behind the tile's last key: nobody joins this split
    // (64 bits: where a sequence takes fewer splits than are launched the others' starts lie
    // at several times its length)
    if (split > 0 && static_cast<int64_t>(split) * span >= vmax) return;
  }
  const int first = split * span_blocks;  // blocks from 0, or of the list

  // Q as the B operand: column l % 16, 16 bytes of each 64-byte half
  v4i_d qf[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  float cs = 0.0f;
  if (live) {
    const int8_t *q = a.q8 + row * a.ldq + (kvh * group_heads + g) * HD + 16 * quarter;
    qf[0] = *reinterpret_cast<const v4i_d *>(q);
    qf[1] = *reinterpret_cast<const v4i_d *>(q + 64);
    cs = a.qs[row * a.ldqs + (kvh * group_heads + g) * a.qs_col] * a.qk_scale * kLog2e;
  }

  const bool once = ONCE || (!LIST && cols <= FEW_COLS);  // (a sequence of one tile)
  uint8_t *const stages = lds.stage + wave * FEW_WAVE;
  const int r8 = lane >> 3, ch = lane & 7;
  const int64_t lane_k = r8 * a.pool.row_bytes + 16 * (ch ^ r8);
  const int64_t lane_v = r8 * a.pool.row_bytes + 16 * (ch ^ (r8 & 3));
  const int64_t lane_v4 = r8 * a.pool.row_bytes + 16 * (ch ^ ((r8 & 3) | 4));

  auto issue = [&](int page, int t0, uint8_t *st) {
    const int64_t at = page * a.pool.page_bytes + t0 * a.pool.row_bytes + kvh * HD;
    const int8_t *k = a.pool.k + at, *v = a.pool.v + at;
    const int64_t eight = 8 * a.pool.row_bytes;
    auto copy = [&](auto nt_tag) {
      constexpr bool NT = decltype(nt_tag)::value;
#pragma unroll
      for (int q = 0; q < 4; ++q) lds_copy16<NT>(k + q * eight + lane_k, stages + FEW_K + q * 1024);
#pragma unroll
      for (int q = 0; q < 4; ++q) lds_copy16<NT>(v + q * eight + (q < 2 ? lane_v : lane_v4), st + FEW_V + q * 1024);
    };
    if (once)
      copy(std::true_type{});
    else
      copy(std::false_type{});
    const int64_t sat = page * a.pool.spage + (t0 + (lane & 31)) * a.pool.srow + kvh;
    lds_copy4((lane < 32 ? a.pool.ks : a.pool.vs) + sat, st + FEW_S);
  };

  float m = -INFINITY, l = 0.0f;
  v4f o[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  int buf = 0;
  for (int part = 0; part < span_blocks; part += FEW_BLOCKS) {
    if constexpr (!LIST) {
      if ((first + part) * KB >= vmax) break;
    }
    // Lane i names the wave's block i of this part: its page, its place there, its first key.
    int bpage = -1, bkey = 0, bt = 0;
    const int nth_block = part + lane * FEW_WAVES + wave;
    if (nth_block < span_blocks) {
      const int per_page = pt / KB;
      const int b = first + nth_block;
      const int nth = b / per_page;
      bt = (b % per_page) * KB;
      if constexpr (LIST) {
        if (nth < a.n_sel) {
          const int id = a.ids[row0 * a.ld_ids + static_cast<int64_t>(kvh) * a.n_sel + nth];
          // a page of the row's: its first key is seen, so it lies in the table
          if (vmax > 0 && id >= 0 && id <= (vmax - 1) / pt) {
            bkey = id * pt + bt;
            if (bkey < vmax) bpage = seq_page(a.seqs, a.pool, seq, id);
          }
        }
      } else {
        bkey = b * KB;
        if (bkey < vmax) bpage = seq_page(a.seqs, a.pool, seq, nth);
      }
    }
    uint64_t todo = __ballot(bpage >= 0);
    auto next = [&]() {  // starts the next block's copies; -1: there is none
      if (todo == 0) return -1;
      const int i = __builtin_ctzll(todo);
      todo &= todo - 1;
      // the reads of this block's K, and of the block before, have been used
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(__builtin_amdgcn_readlane(bpage, i), __builtin_amdgcn_readlane(bt, i), stages + buf * FEW_STAGE);
      return i;
    };
    int ahead = next();  // the block in flight
    while (ahead >= 0) {
      const int now = ahead;
      uint8_t *const st = stages + buf * FEW_STAGE;
      buf ^= 1;
      wait_copies<0>();

      // S^T of two 16-key tiles: lane holds keys 4 quarter + i of each
      float x[8], vsc[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint8_t *kr = stages + FEW_K + (t * 16 + col) * HD;
        const v4i_d k0 = *reinterpret_cast<const v4i_d *>(kr + 16 * (quarter ^ (col & 7)));
        const v4i_d k1 = *reinterpret_cast<const v4i_d *>(kr + 16 * ((4 + quarter) ^ (col & 7)));
        v4i_d s = {0, 0, 0, 0};
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(k0, qf[0], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(k1, qf[1], s, 0, 0, 0);
        const v4f ks = *reinterpret_cast<const v4f *>(st + FEW_S + 4 * (t * 16 + 4 * quarter));
        const v4f vs = *reinterpret_cast<const v4f *>(st + FEW_S + 4 * (KB + t * 16 + 4 * quarter));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[4 * t + i] = static_cast<float>(s[i]) * ks[i] * cs;
          vsc[4 * t + i] = vs[i];
        }
      }
      ahead = next();
      const int key0 = __builtin_amdgcn_readlane(bkey, now);
      const bool edge = key0 + KB > vmin;  // some column does not see the whole block
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + (j >> 2) * 16 + 4 * quarter + (j & 3) >= sees) x[j] = -INFINITY;
      }
      float mb = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      mb = fmaxf(col_max(mb), m);
      const float base = mb == -INFINITY ? 0.0f : mb;
      if (__ballot(mb != m)) {
        const float alpha = exp2_from(m, base);
        l *= alpha;
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] *= alpha;
        m = mb;
      }
      float pv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = exp2_from(x[j], base);
        l += e;
        pv[j] = e * vsc[j];
      }
      if (edge) {  // a scale behind the sequence's end may be anything
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + (j >> 2) * 16 + 4 * quarter + (j & 3) >= sees) pv[j] = 0.0f;
      }
      const Bf16x3 pb = split_bf16(pv);

      // the key that this lane's address names for the transposing read: the 16
      // lanes of a row take 8 keys, two halves of a 16-byte chunk each
      const int rj = (lane & 15) >> 1;
      const int key = 4 * quarter + (rj & 3) + 16 * (rj >> 2);
      const uint8_t *vq = st + FEW_V + key * HD + 8 * (lane & 1);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const v2i_d w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<lds_v2i_ptr_d>(to_lds(vq + 16 * (t ^ vswz(key)))));
        const v8bf vt = int8_bf16(w);
#pragma unroll
        for (int u = 0; u < 3; ++u) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, pb.part[u], o[t], 0, 0, 0);
      }
    }
  }

  // join the waves: each column's rows of O by wave, and (m, l)
  l = col_sum(l);
  __syncthreads();  // every wave is done with its stages
  float *join = reinterpret_cast<float *>(lds.stage);
#pragma unroll
  for (int t = 0; t < 8; ++t)
    *reinterpret_cast<v4f *>(join + (wave * FEW_COLS + col) * FEW_ROW + 16 * t + 4 * quarter) = o[t];
  if (quarter == 0) lds.m[wave][col] = m, lds.l[wave][col] = l;
  __syncthreads();
  const int jc = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
  const int cc = tile * FEW_COLS + jc;
  if (cc >= cols) return;
  float top = lds.m[0][jc];
#pragma unroll
  for (int w = 1; w < FEW_WAVES; ++w) top = fmaxf(top, lds.m[w][jc]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < FEW_WAVES; ++w) {
    const float f = exp2_from(lds.m[w][jc], base);
    sum += f * lds.l[w][jc];
    const float *src = join + (w * FEW_COLS + jc) * FEW_ROW + d0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] += f * src[i];
  }
  // (no key at all: zeros; scores that are all NaN leave a sum of NaN)
  const int jrow = LIST ? row0 : row0 + cc / group_heads;
  const int jhead = kvh * group_heads + (LIST ? cc : cc % group_heads);
  if (whole) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = sum == 0.0f ? 0.0f : r[i] / sum;
    store_row8(a, jrow, jhead, d0, r);
    return;
  }
  const int64_t slot = LIST || p.by_row ? static_cast<int64_t>(jrow) * a.heads + jhead
                                : (static_cast<int64_t>(seq) * a.kv_heads + kvh) * p.most + cc;
  const int64_t at = slot * p.part.splits + split;
  v4f *dst = reinterpret_cast<v4f *>(p.part.o + at * HD + d0);
  dst[0] = v4f{r[0], r[1], r[2], r[3]};
  dst[1] = v4f{r[4], r[5], r[6], r[7]};
  if (d0 == 0) p.part.ml[at] = make_float2(top, sum);
}

// ---- many columns: 128 to a tile -----------------------------------------------
//
// A workgroup takes one tile of 128 columns and one KV head; each of its four waves
// has 32 columns, and all share the keys, 32 a step.  K [32][128] goes to the K
// operand's LDS image as it is; V int8 is turned once for all waves into the 16-bit
// image of the A operand of V^T P^T (a quarter of it by each wave: a transposing read
// hands a lane 8 keys of one channel, in the order in which P's keys lie in the
// registers).  A wave works on a step's values beside the next step's products,
// whose operands have nothing in common, and the copies of four steps are in LDS or
// in flight: one barrier a step.
//
// A matrix instruction takes 33 cycles of its SIMD, under which four to five vector
// instructions go for nothing; each further one costs 2.5, a conversion, a packing or
// a maximum of three 4.5 and an exponential 8.4 (measured).  So the number of vector
// instructions counts as much as that of the 20 matrix ones a step: two terms of P
// instead of three, keys' scales in the scores but the column's in the exponent's FMA,
// a reference that moves by steps of 2^4, whole steps without a mask in a loop of
// their own, integer scores read as floats.  A wave's step is some 700 cycles of vector
// and 660 of matrix instructions and takes 1800 of its SIMD: what a step waits
// beyond its issue is the barrier and the LDS reads.  Three prompts of 1700 rows, 32
// heads on 8: 128 to 138 us from run to run, 0.37 to 0.40 of the rate of a large bf16
// matrix product for the products that the causal mask leaves.  Matrix and vector
// instructions set apart by hand, a wave's priority over its products, 64 keys a step,
// eight waves that halve the keys and a third workgroup a CU (spills) were not faster.
//
// P: where the split's V scales lie within a factor of 2^8 of each other (none is zero,
// or all are) p * vs fits two f16 numbers, with a reference that puts the largest p times the largest vs at
// 2^10 .. 2^15, so the key of the largest p at 2^2 or above: 22 bits from 2^-3 up, and
// below nothing is off by more than 2^-25, 2^-27 of that key (n such keys by n 2^-27 in all;
// sums of n f32 numbers may be off by n 2^-24).  Otherwise the three bf16
// numbers of the 16-column kernel, with a third more time (three prompts of 1700 rows
// 207 us instead of 151, captured, where int8 results take 144).
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int WIDE_COLS = 128;
constexpr int WIDE_SLOTS = 512;    // workgroups at a time, two a CU
constexpr int WIDE_KEYS = KB;      // of a step
constexpr int WIDE_WAVES = 4;
constexpr int WIDE_DEPTH = 4;      // steps whose K and V lie in LDS or on their way
constexpr int WIDE_RING = 256;     // steps whose blocks' places lie in LDS
// Keys of a split at least: 256 rows behind 4000 keys 512: 45 us, 384: 41, 256: 39; 20
// sequences of 1 .. 300 rows at up to 3000 keys 32, 32, 35.
constexpr int WIDE_LEAST = 384;
constexpr int WIDE_OROW = 32 + 4;  // floats of a column's row where the results turn
constexpr float WIDE_ROOM = 4.0f;  // P may reach 2^4 of its reference before O is scaled down

struct WidePlan {
  Partials part;  // slots: (tile, KV head, column)
  int64_t tiles;  // at most
  int least;      // columns of a sequence that are taken here
};

// Key r's 16-byte chunk c of V lies at chunk c ^ vswz_wide(r): the 8 keys of a
// transposing read (two runs of four, 8 apart) meet 8 chunks.
__device__ __forceinline__ int vswz_wide(int key) { return (key & 3) | ((key >> 1) & 4); }

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += static_cast<int>(lane_xor_m(static_cast<uint32_t>(x), d));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x = max(x, static_cast<int>(lane_xor_m(static_cast<uint32_t>(x), d)));
  return __builtin_amdgcn_readfirstlane(x);
}

// The sequence of the unit-th tile of 128 columns, -1 behind the last, and which of
// its tiles it is: tiles are counted 64 sequences at a time, one per lane.  *span:
// the keys of a split, no fewer than the work for each of WIDE_SLOTS workgroups and an
// eighth, so that ragged tiles' splits are no more than the slots either: one more starts
// only when another has ended (4 sequences of 300 rows behind 1000 keys, 32 heads on 8: 74
// us without the eighth, a sixteenth 73, an eighth 67, a quarter 69; 2048 rows 68, 64, 60,
// 56; 512 rows behind 16000 keys 129, 129, 135, 134).
__device__ __forceinline__ int wide_tile(const SeqAttnArgs &a, const WidePlan &p, int unit, int *nth, int *span, SeqSpan *seq) {
  const int lane = threadIdx.x & 63;
  const int group_heads = a.heads / a.kv_heads;
  int found = -1;
  float steps = 0.0f;
  for (int b = 0; b < a.seqs.n_seq; b += 64) {
    int tiles = 0;
    SeqSpan sp{0, 0, 0};
    if (b + lane < a.seqs.n_seq) {
      sp = seq_span(a.seqs, b + lane);
      const int cols = sp.n * group_heads;
      tiles = cols < p.least ? 0 : (cols + WIDE_COLS - 1) / WIDE_COLS;
      const int keys = a.causal ? max(sp.kv - sp.n / 2, 0) : sp.kv;
      steps += static_cast<float>(tiles) * static_cast<float>(keys / WIDE_KEYS + 1);
    }
    if (found >= 0) continue;
    const int total = wave_sum(tiles);
    if (unit < total) {
      // Each sequence's r-th tile from its end comes before any's (r + 1)-th: the last
      // rows see the most keys, and long tiles are to start first.  r is the largest
      // number of rounds that are over before this unit.
      int r = 0;
      for (int bit = 31 - __builtin_clz(wave_max(tiles)); bit >= 0; --bit) {
        const int to = r | (1 << bit);
        if (wave_sum(min(tiles, to)) <= unit) r = to;
      }
      const int k = unit - wave_sum(min(tiles, r));  // the k-th sequence with more than r tiles
      const uint64_t left = __ballot(tiles > r);
      const bool is = tiles > r && __popcll(left & ((1ull << lane) - 1)) == k;
      const int at = __builtin_ctzll(__ballot(is));
      *nth = __builtin_amdgcn_readlane(tiles, at) - 1 - r;
      *seq = {__builtin_amdgcn_readlane(sp.r0, at), __builtin_amdgcn_readlane(sp.n, at), __builtin_amdgcn_readlane(sp.kv, at)};
      found = b + at;
    }
    unit -= total;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) steps += __uint_as_float(lane_xor_m(__float_as_uint(steps), d));
  const float each = steps * static_cast<float>(a.kv_heads) * 1.125f / WIDE_SLOTS;
  const int even = static_cast<int>(ceilf(fminf(each, static_cast<float>(1 << 25)))) * WIDE_KEYS;
  *span = __builtin_amdgcn_readfirstlane(max(split_span(found < 0 ? 0 : seq->kv, p.part.splits, WIDE_LEAST, WIDE_KEYS), even));
  return found;
}

// The most keys that a column of a tile sees.
__device__ __forceinline__ int tile_keys(const SeqAttnArgs &a, const SeqSpan &sp, int col0, int cols) {
  const int group_heads = a.heads / a.kv_heads;
  return a.causal ? max(sp.pos(sp.r0 + (min(cols, col0 + WIDE_COLS) - 1) / group_heads) + 1, 0) : sp.kv;
}

struct WideLds {
  struct Stages {
    uint8_t vt[2][WIDE_KEYS * HD * 2];
    uint8_t k[WIDE_DEPTH][WIDE_KEYS * HD];
    uint8_t v8[WIDE_DEPTH][WIDE_KEYS * HD];
  };
  static_assert(sizeof(Stages) >= 4 * 32 * WIDE_OROW * 4, "the results fit where the steps were");
  __align__(16) Stages st;
  __align__(16) float sc[2 * WIDE_DEPTH][2 * WIDE_KEYS];  // of a step's block ks, then vs
  int2 block[WIDE_RING];                                  // of step % WIDE_RING: page, first token
  uint32_t range[2];
};

__device__ void wide_columns(const SeqAttnArgs &a, const WidePlan &p, int block, WideLds &lds) {
  WideLds::Stages &st = lds.st;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int half = lane >> 5, n32 = lane & 31;
  const int group_heads = a.heads / a.kv_heads;

  const int kvh = block % a.kv_heads;
  const int us = block / a.kv_heads;
  // (split by split: a CU is fed in turn, whether the one before had work or not)
  const int unit = us % static_cast<int>(p.tiles), split = us / static_cast<int>(p.tiles);
  int nth, span;
  SeqSpan sp;
  const int seq = wide_tile(a, p, unit, &nth, &span, &sp);
  if (seq < 0) return;
  const int cols = sp.n * group_heads;
  const int pt = a.pool.page_tokens;
  const int col0 = nth * WIDE_COLS;
  const int c = col0 + wave * 32 + n32;
  const bool live = c < cols;
  const int row = sp.r0 + c / group_heads, head = kvh * group_heads + c % group_heads;
  const int sees = !live ? 0 : a.causal ? max(sp.pos(row) + 1, 0) : sp.kv;
  // the fewest and the most keys that a column sees: the first row's, the last's
  const int first_row = sp.r0 + col0 / group_heads;
  const int tile_min = a.causal ? max(sp.pos(first_row) + 1, 0) : sp.kv;
  const int tile_max = tile_keys(a, sp, col0, cols);
  if (split > 0 && split * static_cast<int64_t>(span) >= tile_max) return;
  const int first = split * span, end = min(tile_max, first + span);
  const int steps = (end - first + WIDE_KEYS - 1) / WIDE_KEYS;  // <= 0: none

  v4i_d qf[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = v4i_d{0, 0, 0, 0};
  float cs = 0.0f;
  if (live) {
    const int8_t *q = a.q8 + row * a.ldq + head * HD + 16 * half;
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const v4i_d *>(q + 32 * i);
    cs = a.qs[row * a.ldqs + head * a.qs_col] * a.qk_scale * kLog2e;
  }

  auto place = [&](int step) {
    const int key = first + step * WIDE_KEYS;
    return make_int2(seq_page(a.seqs, a.pool, seq, key / pt), key % pt);
  };

  // Copies: wave w takes keys 8 w .. 8 w + 7 of a step (of block w / 4).
  const int r8 = lane >> 3, ch = lane & 7;
  const int64_t my_row = (8 * wave + r8) * a.pool.row_bytes + kvh * HD;
  const int64_t lane_k = my_row + 16 * (ch ^ r8), lane_v = my_row + 16 * (ch ^ vswz_wide(8 * wave + r8));
  auto copy = [&](int step) {
    int2 at = lds.block[step % WIDE_RING];
    at = make_int2(__builtin_amdgcn_readfirstlane(at.x), __builtin_amdgcn_readfirstlane(at.y));
    if (at.x < 0) return;
    const int64_t bytes = at.x * a.pool.page_bytes + at.y * a.pool.row_bytes;
    lds_copy16(a.pool.v + bytes + lane_v, st.v8[step % WIDE_DEPTH] + wave * 8 * HD);
    lds_copy16(a.pool.k + bytes + lane_k, st.k[step % WIDE_DEPTH] + wave * 8 * HD);
    if (wave == 0)
      lds_copy4((half ? a.pool.vs : a.pool.ks) + at.x * a.pool.spage + (at.y + n32) * a.pool.srow + kvh, lds.sc[step % (2 * WIDE_DEPTH)]);
  };

  // The blocks' places, and the range of the V scales' magnitudes (as integers), 32 lanes
  // a block: of the whole split, its start last, beside whose scales
  // the first steps' copies are under way.
  bool missing = false;
  uint32_t most = 0, least = 0x7f800000u;
  if (tid < 2) lds.range[tid] = tid == 0 ? most : least;
  for (int part = (max(steps, 1) - 1) / WIDE_RING * WIDE_RING;; part -= WIDE_RING) {
    const int n = min(steps - part, WIDE_RING);
    bool hole = false;
    if (tid < n) {
      const int2 at = place(part + tid);
      hole = at.x < 0;
      lds.block[tid] = at;
    }
    missing |= __syncthreads_or(hole) != 0;
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < WIDE_DEPTH; ++i)
        if (i < steps) copy(i);
    }
#pragma unroll 4
    for (int i = tid >> 5; i < n; i += 2 * WIDE_WAVES) {
      const int2 at = lds.block[i];
      if (at.x >= 0 && first + (part + i) * KB + n32 < end) {
        const uint32_t v = __float_as_uint(a.pool.vs[at.x * a.pool.spage + (at.y + n32) * a.pool.srow + kvh]) & 0x7fffffffu;
        most = max(most, v);
        least = min(least, v);
      }
    }
    if (part == 0) break;
    __syncthreads();
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    most = max(most, lane_xor_m(most, d));
    least = min(least, lane_xor_m(least, d));
  }
  if (lane == 0) {
    atomicMax(&lds.range[0], most);
    atomicMin(&lds.range[1], least);
  }
  wait_copies<0>();
  lds_barrier();
  most = __builtin_amdgcn_readfirstlane(lds.range[0]), least = __builtin_amdgcn_readfirstlane(lds.range[1]);
  // Narrow: within a factor of 2^8, and no closer to the ends than 2^64, or all zeros.  A
  // zero beside others is not: its key may have the largest score, far below which the
  // others' products would leave f16.
  const int expo = static_cast<int>(most >> 23) - 127;
  const bool narrow = most == 0 || (expo >= -64 && expo <= 64 && least >= most - (8u << 23));
  // with p = 2^(x - top + lift) p vs < 2^11 at the largest x
  const float lift = narrow && most ? static_cast<float>(10 - expo) : 0.0f;

  // The softmax's reference, a score but for the column's scale, at most WIDE_ROOM (base 2)
  // short of the largest, so that O is scaled down a few times in all, not at every new
  // maximum.  Exponents are (x - ref) * size + lift: the reference's own is exactly lift,
  // however large it is.  While no reference of the wave is beyond 2^10 (`far`) x * size + add
  // is as good and an instruction less (three prompts of 1700 rows 134.5 us without it, 131.3
  // with); add's rounding at 2^26 would be more than f16 has room for.
  // room: the exponent at which ref moves, -inf until there is a score; those of -inf never are
  // the reference, and have no weight.
  float ref = 0.0f, room = -INFINITY, add = lift, l = 0.0f;
  bool far = false;
  v16f o[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
  const float size = fabsf(cs), sign = __builtin_copysignf(1.0f, cs);
  const bool turned = __ballot(cs < 0.0f) != 0;  // some column's scale is negative

  // S of a step, |S| <= 2^21, on top of the bits of 1.5 * 2^23: as f32, that plus S (a
  // subtraction then instead of a conversion, which takes twice its time).
  constexpr int kOnTop = 0x4B400000;
  v16i on_top;
#pragma unroll
  for (int i = 0; i < 16; ++i) on_top[i] = kOnTop;
  asm volatile("" : "+v"(on_top));  // kept in registers, not made anew in every step
  auto products = [&](const v4i_d (&kf)[4], v16i &s) {
    s = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[0], qf[0], on_top, 0, 0, 0);
#pragma unroll
    for (int i = 1; i < 4; ++i) s = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[i], qf[i], s, 0, 0, 0);
  };
  auto keys_of = [&](int step, v4i_d (&kf)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      kf[i] = *reinterpret_cast<const v4i_d *>(st.k[step % WIDE_DEPTH] + n32 * HD + 16 * ((2 * i + half) ^ (n32 & 7)));
  };

  // Their scores but for the column's scale: register i is key 8 (i / 4) + 4 half +
  // i % 4.  EDGE: some column does not see some key, or has a negative scale; `seen`
  // keeps which, since nothing of that key may enter the sums, not even a scale's NaN.  Returns the
  // column's largest.
  float x[16];
  uint32_t seen = ~0u;
  auto scores = [&](int step, const v16i &s, auto edge_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f ks = *reinterpret_cast<const v4f *>(lds.sc[step % (2 * WIDE_DEPTH)] + 8 * i + 4 * half);
      if constexpr (EDGE) {
        if (turned) ks *= sign;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = (__int_as_float(s[4 * i + j]) - __int_as_float(kOnTop)) * ks[j];
    }
    seen = ~0u;
    if constexpr (EDGE) {
      seen = 0;
      const int limit = lds.block[step % WIDE_RING].x < 0 ? 0 : sees - (first + step * WIDE_KEYS + 4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = 8 * (i >> 2) + (i & 3) < limit;
        seen |= static_cast<uint32_t>(in) << i;
        if (!in) x[i] = -INFINITY;
      }
    }
    float mb = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mb = fmaxf(mb, x[i]);
    const LanePair pr = lane_pair32(__float_as_uint(mb));
    return fmaxf(__uint_as_float(pr.a), __uint_as_float(pr.b));
  };
  auto exponent = [&](float score, auto edge_tag) {
    return decltype(edge_tag)::value ? __builtin_fmaf(score - ref, size, lift) : __builtin_fmaf(score, size, add);
  };
  auto refer = [&](float top, auto edge_tag) {
    const bool up = top > -INFINITY && !(exponent(top, edge_tag) <= room);
    if (__ballot(up)) {
      const float to = up ? top : ref;
      const float alpha = room == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ref - to) * size);
      l *= alpha;
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] *= alpha;
      ref = to;
      add = __builtin_fmaf(-ref, size, lift);
      far = __ballot(!(fabsf(add) < 0x1p+10f)) != 0;
      if (up) room = lift + WIDE_ROOM;
    }
  };

  // P of 16 keys (registers 8 r .. 8 r + 7) times their V scales, in the terms that
  // the matrix cores take.
  auto weights = [&](int step, int r, auto edge_tag, auto narrow_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    const float *vs = lds.sc[step % (2 * WIDE_DEPTH)] + KB + 16 * r + 4 * half;
    const v4f va = *reinterpret_cast<const v4f *>(vs), vc = *reinterpret_cast<const v4f *>(vs + 8);
    float e[8], pv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(exponent(x[8 * r + j], edge_tag));
      const bool in = !EDGE || (seen >> (8 * r + j) & 1);
      if (!in) e[j] = 0.0f;
      pv[j] = e[j] * (j < 4 ? va[j] : vc[j - 4]);
      if (!in) pv[j] = 0.0f;
    }
    l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    if constexpr (decltype(narrow_tag)::value)
      return split_f16(pv);
    else
      return split_bf16(pv);
  };
  auto values = [&](int step, int r, const auto &pb) {
    const uint8_t *vt = st.vt[step & 1] + (r * 4 * 64 + lane) * 16;
    if constexpr (std::is_same_v<std::decay_t<decltype(pb)>, F16x2>) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const v8h *>(vt + t * 1024), pb.part[u], o[t], 0, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 3; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const v8bf *>(vt + t * 1024), pb.part[u], o[t], 0, 0, 0);
    }
  };

  // This wave's quarter of a step's V: channels 32 wave .. + 31.
  const int vj = (lane & 15) >> 1;
  const int vkey = 8 * (vj >> 2) + 4 * half + (vj & 3);
  auto turn = [&](int step, auto narrow_tag) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int key = 16 * r + vkey, chunk = 2 * wave + ((lane >> 4) & 1);
      const uint8_t *src = st.v8[step % WIDE_DEPTH] + key * HD + 16 * (chunk ^ vswz_wide(key)) + 8 * (lane & 1);
      const v2i_d w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<lds_v2i_ptr_d>(to_lds(src)));
      uint8_t *dst = st.vt[step & 1] + ((r * 4 + wave) * 64 + lane) * 16;
      if constexpr (decltype(narrow_tag)::value)
        *reinterpret_cast<v8h *>(dst) = int8_f16(w);
      else
        *reinterpret_cast<v8bf *>(dst) = int8_bf16(w);
    }
  };

  int step = 0;
  auto run = [&](int to, auto edge_tag, auto narrow_tag) {
    for (; step < to; ++step) {
      if (!decltype(edge_tag)::value && far) break;  // (to the other loop)
      if (step % (WIDE_RING / 2) == 0 && step > 0) {  // the places after the next, over those gone by
        const int next = step + WIDE_RING / 2 + tid;
        if (tid < WIDE_RING / 2 && next < steps) lds.block[next % WIDE_RING] = place(next);
      }
      const bool more = !decltype(edge_tag)::value || step + 1 < steps;
      if (step + WIDE_DEPTH < steps) copy(step + WIDE_DEPTH);
      v16i s;
      v4i_d kf[4];
      if (more) keys_of(step + 1, kf);
      const auto p0 = weights(step, 0, edge_tag, narrow_tag);
      if (more) products(kf, s);
      const auto p1 = weights(step, 1, edge_tag, narrow_tag);
      values(step, 0, p0);
      if (more) turn(step + 1, narrow_tag);
      values(step, 1, p1);
      if (more) refer(scores(step + 1, s, edge_tag), edge_tag);
      // the step after next is needed now; those behind it may be on their way, as
      // many copies as a wave issues for them (fewer where a page is missing)
      if (missing || step + WIDE_DEPTH >= steps)
        wait_copies<0>();
      else if (wave == 0)
        wait_copies<3 * (WIDE_DEPTH - 2)>();
      else
        wait_copies<2 * (WIDE_DEPTH - 2)>();
      lds_barrier();
    }
  };
  auto all = [&](auto narrow_tag) {
    turn(0, narrow_tag);
    v16i s;
    v4i_d kf[4];
    keys_of(0, kf);
    products(kf, s);
    refer(scores(0, s, std::true_type{}), std::true_type{});
    lds_barrier();
    // Steps that every column sees whole, then the others (all, where a page is
    // missing, a scale negative or a score far from 0): two loops, since one with both forms of a step
    // keeps O twice.
    if constexpr (decltype(narrow_tag)::value)
      run(missing || turned ? 0 : clampi((tile_min - first) / WIDE_KEYS, 0, steps) - 1, std::false_type{}, narrow_tag);
    run(steps, std::true_type{}, narrow_tag);
  };
  if (steps > 0) {
    if (narrow)
      all(std::true_type{});
    else
      all(std::false_type{});
  }

  {
    const LanePair pr = lane_pair32(__float_as_uint(l));
    l = __uint_as_float(pr.a) + __uint_as_float(pr.b);
  }
  const bool whole = tile_max <= span;
  const int64_t at = whole || !live ? 0 : ((static_cast<int64_t>(unit) * a.kv_heads + kvh) * WIDE_COLS + c - col0) * p.part.splits + split;
  // (a partial result without its lift, a power of two that the other splits do not share)
  const float inv = !whole ? __builtin_amdgcn_exp2f(-lift) : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int t = 0; t < 4; ++t) o[t] *= inv;
  if (!whole && live && half == 0) p.part.ml[at] = make_float2(room == -INFINITY ? -INFINITY : ref * size, l * inv);
  if (whole && a.o8) {
    float pk = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) pk = fmaxf(pk, fabsf(o[t][i]));
    const LanePair pr = lane_pair32(__float_as_uint(pk));
    const float scale = __fmul_rn(fmaxf(__uint_as_float(pr.a), __uint_as_float(pr.b)), inv127());
    if (!live) return;
    const double y = rcp64(scale);
    int8_t *dst = a.o8 + row * a.ldo8 + head * HD;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        dst[32 * t + 8 * (i >> 2) + 4 * half + (i & 3)] = static_cast<int8_t>(quant_rcp(o[t][i], y));
    if (half == 0) a.os[row * a.ldos + head * a.os_col] = scale;
    return;
  }
  // f32 rows through LDS (the steps' last barrier is behind every wave, and a wave
  // keeps to its own part), 32 channels at a time:
  // written in 128-byte pieces
  float *const turn_row = reinterpret_cast<float *>(&st) + wave * 32 * WIDE_OROW;
  const int64_t mine = !live ? -1 : whole ? row * a.ldo + head * HD : at * HD;
  float *const to = whole ? a.out : p.part.o;
  const bool words = !whole || a.out_words;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<v4f *>(turn_row + n32 * WIDE_OROW + 8 * i + 4 * half) = v4f{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t off = __shfl(mine, 8 * k + r8);
      const v4f r = *reinterpret_cast<const v4f *>(turn_row + (8 * k + r8) * WIDE_OROW + 4 * ch);
      if (off < 0) continue;
      float *dst = to + off + 32 * t + 4 * ch;
      if (words) {
        *reinterpret_cast<v4f *>(dst) = r;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = r[i];
      }
    }
  }
}

// ---- launches -------------------------------------------------------------------

template <bool LIST, bool ONCE>
__global__ void __launch_bounds__(256, 3) seq_attn_few_kernel(SeqAttnArgs a, FewPlan p) {
  __shared__ FewLds lds;
  few_columns<LIST, ONCE>(a, p, blockIdx.x, lds);
}

// Both kinds of sequences in one launch, so that short ones fill the CUs beside the
// long ones: the first `wide` workgroups take the 128-column tiles.
__global__ void __launch_bounds__(256, 2) seq_attn_mixed_kernel(SeqAttnArgs a, FewPlan fp, WidePlan wp, int wide) {
  __shared__ union Lds {
    FewLds few;
    WideLds wide;
  } lds;
  if (static_cast<int>(blockIdx.x) < wide)
    wide_columns(a, wp, blockIdx.x, lds.wide);
  else
    few_columns<false, true>(a, fp, blockIdx.x - wide, lds.few);
}

// Joins the splits of slots: 16 lanes of 8 channels a slot, of many splits 16 such
// groups over the splits in turn (GROUPS; 16 slots a workgroup otherwise): 4 to 5 us,
// most of it the launch.  A cell is what slots are counted in: (sequence, KV head) or
// row of the 16-column kernel, (tile, KV head) of the 128-column one.
struct JoinLds {
  float o[4][HD], sum[4];
};

template <int GROUPS, bool WIDE, class Plan>
__device__ void join_slots(const SeqAttnArgs &a, const Plan &plan, int cell_cols, int block, JoinLds &lds) {
  const Partials &p = plan.part;
  constexpr int PER = 16 / GROUPS;
  const int group = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
  const int blocks = (cell_cols + PER - 1) / PER;
  const int cell = block / blocks;
  const int c = block % blocks * PER + (GROUPS == 1 ? group : 0);  // column of the cell
  const int group_heads = a.heads / a.kv_heads;
  int row, head, n;
  if (!WIDE && a.ids) {
    row = cell, head = c;
    if (row_at(a.seqs, row).seq < 0 || c >= a.heads) return;
    n = p.splits;
  } else {
    int col = c, cols, seq, span;
    SeqSpan sp;
    if constexpr (WIDE) {
      int nth;
      seq = wide_tile(a, plan, cell / a.kv_heads, &nth, &span, &sp);
      if (seq < 0) return;
      cols = sp.n * group_heads;
      if (tile_keys(a, sp, nth * WIDE_COLS, cols) <= span) return;  // written as it is
      col += nth * WIDE_COLS;
    } else {
      seq = cell / a.kv_heads;
      sp = seq_span(a.seqs, seq);
      cols = sp.n * group_heads;
      span = few_span(plan, sp.kv, cols);
      if (cols > plan.most || sp.kv <= span) return;  // elsewhere; written as it is
    }
    if (c >= cell_cols || col >= cols) return;
    row = sp.r0 + col / group_heads;
    head = cell % a.kv_heads * group_heads + col % group_heads;
    const int sees = a.causal ? max(sp.pos(row) + 1, 0) : sp.kv;
    n = (sees + span - 1) / span;
  }
  int64_t slot = static_cast<int64_t>(cell) * cell_cols + c;
  if constexpr (!WIDE) {
    if (plan.by_row) slot = static_cast<int64_t>(row) * a.heads + head;
  }
  const int64_t at = slot * p.splits;
  float top = -INFINITY;
  for (int s = threadIdx.x & 15; s < n; s += 16) top = fmaxf(top, p.ml[at + s].x);
  top = fmaxf(top, lane_xor<1>(top));
  top = fmaxf(top, lane_xor<2>(top));
  top = fmaxf(top, lane_xor<4>(top));
  top = fmaxf(top, lane_xor<8>(top));
  const float base = top == -INFINITY ? 0.0f : top;
  float r[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f;
#pragma unroll 4
  for (int s = GROUPS == 1 ? 0 : group; s < n; s += GROUPS) {
    const float2 ml = p.ml[at + s];
    const float f = exp2_from(ml.x, base);
    sum += f * ml.y;
    const v4f *src = reinterpret_cast<const v4f *>(p.o + (at + s) * HD + d0);
    const v4f u = src[0], v = src[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] += f * u[i], r[4 + i] += f * v[i];
  }
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = col_sum(r[i]);
    sum = col_sum(sum);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < 16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) lds.o[wave][d0 + i] = r[i];
      if (d0 == 0) lds.sum[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= 16) return;
    sum = (lds.sum[0] + lds.sum[1]) + (lds.sum[2] + lds.sum[3]);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (lds.o[0][d0 + i] + lds.o[1][d0 + i]) + (lds.o[2][d0 + i] + lds.o[3][d0 + i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = sum == 0.0f ? 0.0f : r[i] / sum;
  store_row8(a, row, head, d0, r);
}

// 16 groups share a slot from 13 splits on, where slots are few: at many the launch's
// workgroups would cost more than the splits one after another.
constexpr int JOIN_MANY = 12, JOIN_SLOTS = 1024;
__host__ __device__ inline bool join_wide(const Partials &p) { return p.splits > JOIN_MANY && p.slots <= JOIN_SLOTS; }

int join_cols(const SeqAttnArgs &a, const FewPlan &p) { return a.ids ? a.heads : p.most; }
int join_cols(const SeqAttnArgs &, const WidePlan &) { return WIDE_COLS; }

template <class P>
int64_t join_wgs(const SeqAttnArgs &a, const P &plan) {
  const int cols = join_cols(a, plan);
  return plan.part.slots / cols * (join_wide(plan.part) ? cols : (cols + 15) / 16);
}

// The first `few` workgroups join the 16-column kernel's slots.
__global__ void __launch_bounds__(256) seq_attn_join_kernel(SeqAttnArgs a, FewPlan fp, WidePlan wp, int few) {
  __shared__ JoinLds lds;
  const int block = blockIdx.x;
  if (block < few) {
    const int cols = a.ids ? a.heads : fp.most;
    if (join_wide(fp.part))
      join_slots<16, false>(a, fp, cols, block, lds);
    else
      join_slots<1, false>(a, fp, cols, block, lds);
  } else if (join_wide(wp.part)) {
    join_slots<16, true>(a, wp, WIDE_COLS, block - few, lds);
  } else {
    join_slots<1, true>(a, wp, WIDE_COLS, block - few, lds);
  }
}

// ---- plans --------------------------------------------------------------------

constexpr int64_t kMaxGrid = (int64_t(1) << 32) / 256 - 1;  // workgroups of 256 lanes in a launch

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits `keys` at most over workgroups, `units` of which would run without a split,
// until there are about `want` of them: 64 splits at most, of `least` keys or more.  A
// max_kv far above the lengths adds workgroups that end at once, no longer splits: 16 rows
// at 500 .. 2000 keys take 19.5 us with a max_kv of 2000 and of 131072 (26 where the spans
// followed max_kv), 512 rows behind 1500 keys 48 both ways (116).
void plan_splits(int64_t units, int64_t keys, int64_t want, int step, int least, Partials &p) {
  if (keys < 1) keys = 1;
  if (units < 1) units = 1;
  int64_t splits = units >= want ? 1 : want / units;
  if (splits > 64) splits = 64;
  int64_t span = cdiv(cdiv(keys, splits), step) * step;
  if (span < least) span = least;
  p.span = static_cast<int>(span);
  p.splits = static_cast<int>(cdiv(keys, span));
}

// Sequences of up to FEW_MOST columns go to the kernel of 16-column tiles, and all
// of a call do where none has more than FEW_ALL, or while rows x heads x max_kv stays
// small: its tiles fill the CUs sooner.  us, 16-column / 128-column tiles, 16 heads on 8:
// 32 rows behind 500 keys 11 / 24, 512 rows (4.2e6) 18 / 26, 64 rows behind 4000 keys
// (4.2e6) 24 / 29, 8 x 64 rows behind 1000 keys (8.7e6) 31 / 35, 1024 rows (17e6) 29 /
// 34, 256 rows behind 4000 keys (17e6) 45 / 41.  8 sequences behind 4000 keys: of 16 rows
// (32 columns) 32 / 47, 24 (48) 36 / 48, 32 (64) 43 / 48; 64 behind 2000, 64 heads on 8:
// of 4 rows (32) 91 / 124, of 8 (64) 137 / 125.  Beside longer sequences only those of
// one tile: with tiles for 48 columns 60 decoding rows and 4 chunks of 128 rows take 79
// instead of 70.
constexpr int FEW_MOST = 16, FEW_ALL = 48;
constexpr int64_t FEW_PAIRS = 12 << 20;
// Workgroups to split for: equal lists of pages 1024, sequences, whose lengths differ,
// more (64 rows at 500 .. 4000 keys 1024: 62 us, 1536: 56, 2304: 56; 92 rows' lists 49,
// 53, 56).  Splits of one length for all sequences, by the work of the batch: 57.
constexpr int LIST_WANT = 1024, FEW_WANT = 1536, WIDE_WANT = 1536;

struct Plan {
  FewPlan few;
  WidePlan wide;
  bool any_wide;
  int64_t few_held, wide_held;  // partial results
};

Plan plan_attn(const SeqAttnArgs &a) {
  Plan p{};
  const int64_t g = a.heads / a.kv_heads, rows = a.seqs.rows, n_seq = a.seqs.n_seq;
  const int64_t cols = a.ids ? g : a.seqs.max_rows * g;  // of a sequence (listed pages: of a row), at most
  const bool small = rows * a.heads * a.seqs.max_kv <= FEW_PAIRS && n_seq * cdiv(cols, FEW_COLS) * a.kv_heads <= 8 * FEW_WANT;
  p.any_wide = !a.ids && cols > FEW_ALL && !small;
  const int64_t few_cols = p.any_wide ? FEW_MOST : cols < 1 ? 1 : cols;
  p.few.most = static_cast<int>(few_cols);
  p.few.tiles = static_cast<int>(cdiv(few_cols, FEW_COLS));
  p.few.units = (a.ids ? rows : n_seq) * p.few.tiles;
  p.few.each = static_cast<int>(cdiv(FEW_WANT, (n_seq < 1 ? 1 : n_seq) * a.kv_heads));
  plan_splits((a.ids ? p.few.units : n_seq) * a.kv_heads, a.ids ? int64_t(a.n_sel) * a.pool.page_tokens : a.seqs.max_kv,
              a.ids ? LIST_WANT : FEW_WANT, FEW_STEP, FEW_LEAST, p.few.part);
  const int64_t by_row = rows * a.heads, by_col = n_seq * a.kv_heads * few_cols;
  p.few.by_row = !a.ids && by_row < by_col;
  if (p.few.part.splits > 1) {
    p.few.part.slots = a.ids ? by_row : by_col;
    p.few_held = std::min(p.few.part.slots, by_row) * p.few.part.splits;
  }
  if (p.any_wide) {
    p.wide.least = FEW_MOST + 1;
    const int64_t wide_seqs = rows * g / p.wide.least;
    p.wide.tiles = rows * g / WIDE_COLS + (n_seq < wide_seqs ? n_seq : wide_seqs);
    plan_splits(p.wide.tiles * a.kv_heads, a.seqs.max_kv, WIDE_WANT, WIDE_KEYS, WIDE_LEAST, p.wide.part);
    if (p.wide.part.splits > 1) p.wide.part.slots = p.wide.tiles * a.kv_heads * WIDE_COLS;
    p.wide_held = p.wide.part.slots * p.wide.part.splits;
  }
  return p;
}

// The most that units x splits of plan_splits comes to, for up to so many units and keys
// (0: no call of these sizes is split).
int64_t most_splits(int64_t units, int64_t keys, int64_t want, int least) {
  return keys <= least ? 0 : std::min(want, units * std::min<int64_t>(64, cdiv(keys, least)));
}

// The most partial results of any call whose counts are at most these.  Splits fall as
// units grow, so a call's own number rises and falls with its counts.
int64_t most_partials(const SeqAttnArgs &a) {
  const int64_t g = a.heads / a.kv_heads, rows = a.seqs.rows, n_seq = a.seqs.n_seq;
  if (a.ids) {  // units x splits x (heads of a tile)
    const int64_t tiles = cdiv(g, FEW_COLS);
    return cdiv(most_splits(rows * tiles * a.kv_heads, int64_t(a.n_sel) * a.pool.page_tokens, LIST_WANT, FEW_LEAST) * g, tiles);
  }
  const int64_t cols = std::max<int64_t>(1, a.seqs.max_rows * g), keys = a.seqs.max_kv;
  int64_t few = most_splits(n_seq * a.kv_heads, keys, FEW_WANT, FEW_LEAST) * std::min<int64_t>(cols, FEW_ALL);
  // Small calls of more columns, (row, head) slots at most: of more than FEW_LEAST keys, at
  // most FEW_PAIRS / keys of them, each of at most 2 keys / FEW_LEAST splits.
  if (cols > FEW_ALL && few > 0) few = std::max(few, 2 * FEW_PAIRS / FEW_LEAST);
  few = std::min(few, most_splits(rows * a.heads, keys, INT64_MAX, FEW_LEAST));
  const Plan p = plan_attn(a);  // (a call that is small, or of few columns, has none larger below it)
  return few + (p.any_wide ? most_splits(p.wide.tiles * a.kv_heads, keys, WIDE_WANT, WIDE_LEAST) * WIDE_COLS : 0);
}

constexpr uint64_t kPartialBytes = HD * 4 + 8;

}  // namespace

uint64_t seq_attn_ws_bytes(const SeqAttnArgs &a) {
  const Plan p = plan_attn(a);
  return static_cast<uint64_t>(p.few_held + p.wide_held) * kPartialBytes;
}

uint64_t seq_attn_ws_most(const SeqAttnArgs &a) { return static_cast<uint64_t>(most_partials(a)) * kPartialBytes; }

hipError_t launch_seq_attn(const SeqAttnArgs &args, hipStream_t s) {
  if (args.seqs.rows == 0 || args.seqs.n_seq == 0) return hipSuccess;
  SeqAttnArgs a = args;
  a.out_words = a.out && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.ldo & 3) == 0;
  Plan p = plan_attn(a);
  const int64_t nf = p.few_held, nw = p.wide_held;
  p.few.part.o = static_cast<float *>(a.ws);
  p.wide.part.o = p.few.part.o + nf * HD;
  p.few.part.ml = reinterpret_cast<float2 *>(p.wide.part.o + nw * HD);
  p.wide.part.ml = p.few.part.ml + nf;
  const int64_t few = cdiv(p.few.units * p.few.part.splits, 8) * 8 * a.kv_heads;
  const int64_t wide = p.any_wide ? p.wide.tiles * p.wide.part.splits * a.kv_heads : 0;
  if (few + wide > kMaxGrid) return hipErrorInvalidValue;
  static_assert(64 * FEW_WAVES == 256 && 64 * WIDE_WAVES == 256, "one launch shape");
  if (wide)
    hipLaunchKernelGGL(seq_attn_mixed_kernel, dim3(static_cast<unsigned>(wide + few)), dim3(256), 0, s, a, p.few, p.wide,
                       static_cast<int>(wide));
  else if (a.ids && a.seqs.max_rows <= 1)
    hipLaunchKernelGGL((seq_attn_few_kernel<true, true>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, a, p.few);
  else if (a.ids)
    hipLaunchKernelGGL((seq_attn_few_kernel<true, false>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, a, p.few);
  else if (p.few.tiles == 1)
    hipLaunchKernelGGL((seq_attn_few_kernel<false, true>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, a, p.few);
  else
    hipLaunchKernelGGL((seq_attn_few_kernel<false, false>), dim3(static_cast<unsigned>(few)), dim3(256), 0, s, a, p.few);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int64_t join_few = join_wgs(a, p.few), join = join_few + join_wgs(a, p.wide);
  if (join == 0) return hipSuccess;
  if (join > kMaxGrid) return hipErrorInvalidValue;
  hipLaunchKernelGGL(seq_attn_join_kernel, dim3(static_cast<unsigned>(join)), dim3(256), 0, s, a, p.few, p.wide,
                     static_cast<int>(join_few));
  return hipGetLastError();
}

}  // namespace q3
