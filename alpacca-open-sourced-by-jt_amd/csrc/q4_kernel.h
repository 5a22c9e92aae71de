// Attention over a page pool of 4-bit codes, for one token of a sequence or a
// run of them.
//
// Sequence b holds prefix_lens[b] rows and behind them one row for each of
// its counts[b] tokens; token i sees the rows up to and with its own:
//   out[b, i, h] = softmax_j(scale * q[b, i, h] . K[j, h / G]) . V[j, h / G],
//   j <= prefix + i, K and V = least + step * code,
// times sigmoid(gate) where given.  Tokens at or past counts[b], and those
// whose row lies past `length`, give zeros.
//
// The matrix products run on the codes themselves.  With g the groups of 32
// channels, c the codes, d the steps and m the least values,
//   q . k_j   = sum_g d_jg (q_g . c_jg) + m_jg (sum of q_g),
//   sum_j p_j v_j = (sum_j (p_j d_jg) (c_jg - 8)) + (sum_j p_j (m_jg + 8 d_jg)):
// a product of 32 channels per group, its result times a step per key; and
// probabilities times steps against the codes, with least values and steps as
// one more small product (whose rows of ones give the sum of p).
//
// A code is the float16 number c 2^-24 as its bits stand, a subnormal that the
// matrix unit takes at full rate, so a word of eight codes becomes an operand
// in five instructions; codes that stay four bits up count 16-fold, which q
// takes back.  The unit's sums of such products are coarser than float32, which
// the scores of 16-bit queries bear: fp16 results, before their own rounding,
// are 1.5e-6 off where scores have deviation 1, 1.2e-5 at 64.  Sums over many
// rows do not: subnormal codes of V cost 1e-5 of the result on 500 rows and
// 1.5e-4 on 131072, with least values that cancel them only at the end 1.6e-5
// and 1.9e-4.  So V's codes, and K's for float32 queries, are centred and made
// normal numbers, (c - 8) 2^-9, by one more instruction a pair, and least + 8
// step joined tile by tile: float32 results are 4e-7 to 6e-7 off on 500 to
// 131072 rows, 1.2e-6 where a wave alone sums 2048 of them (64 x 1 on 8192).
// Values below 1e-3 lose more (p d is subnormal): 1.6e-6 at 1e-4, 1.7e-5 at
// 1e-5.  (4 x 1 on 131072 rows, 32/8 heads of 128, fp16: 140.5 us for 137.)
// Nothing is rounded but q (float32: two float16 parts, 22 bits; others
// exactly) and p d (two parts).
#pragma once

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "alpx_common.h"
#include "prefill_run.h"
#include "q4_internal.h"
#include "row_shares.h"

namespace alpx {
namespace {

typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = kQ4Rows;
constexpr int kWaves = kQ4Waves;
constexpr float kUnit = 0x1p9f;  // a centred code of 1 is 1 / kUnit as an operand
constexpr float kLift = 12.f;   // P is formed 2^12 times as large: float16 keeps
constexpr float kSlack = 3.f;   // more of small ones; its reference may lag by 2^3

// Shape of a kernel: T of q, gate and the arithmetic's precision, G groups of
// 32 channels, CT column tiles of 16 per wave, CP of whose columns are
// queries, TP tiles to a step, a ring of RING steps per wave, blocks per CU.
//
// CP below 16: the 16 columns of a product are CP queries times R = 16 / CP
// groups.  Each of those columns holds its query's channels of its own group
// and zeros elsewhere, so the products of R groups run into one accumulator,
// whose columns then take their own group's steps; a query's score is the sum
// of its columns.  Likewise a column's probabilities take its own group's
// steps, and of V's product with them its own group's channels count.  As many
// products, but a quarter (half) of the multiplications by steps.
template <typename T_, int G_, int CT_, int CP_, int TP_, int RING_, int CU_>
struct Q4Shape {
  typedef T_ T;
  static constexpr int G = G_, CT = CT_, TP = TP_, RING = RING_, D = 32 * G_, kPerCu = CU_;
  static constexpr int CP = CP_, R = 16 / CP_;
  static constexpr bool kPacked = CP < 16;
  static constexpr int NT = (G + R - 1) / R;  // accumulators that the groups' products run into
  static_assert(!kPacked || CT == 1, "one column tile");
  static constexpr int QP = sizeof(T_) == 4 ? 2 : 1;  // parts of q
  static constexpr bool kOnce = CT == 1;  // one column tile: nobody reads a tile twice
  // float32 takes K's codes centred as well.
  static constexpr bool kCentred = QP == 2;
  static constexpr float kSumScale = kCentred ? 0x1p-9f : 0x1p-6f;  // of a group's sum of q, in parts
  static constexpr float kCodeUnit = kCentred ? kUnit : 0x1p24f;  // of K
  static constexpr float kSumUnit = (kPacked ? 1.f : 1.f / kSumScale) / kCodeUnit;  // of the sums of q
  static constexpr int kBases = (G_ + 3) / 4;
  static constexpr int kCols = CP * CT;
  static constexpr int kCodeB = kRows * 16 * G;        // codes of K or V in a tile
  static constexpr int kScaleB = 2 * G * kRows * 2;    // steps, then least values
  static constexpr int kTileB = 2 * (kCodeB + kScaleB);
  static constexpr int kCodeLoads = (kCodeB + 1023) / 1024;
  static constexpr int kStepLoads = TP * (2 * kCodeLoads + 2);
  static constexpr int kStepRows = TP * kRows;
  static constexpr int kStepB = TP * kTileB;
  static constexpr int kMergeRow = D + 4;              // floats
  static constexpr int kMergeB = kWaves * 16 * kMergeRow * 4 + kWaves * 16 * CT * 16;
  static constexpr int kRingB = kWaves * RING * kStepB;
  static constexpr int kLds = kRingB > kMergeB ? kRingB : kMergeB;
  static_assert(kLds * kPerCu <= 160 * 1024, "blocks fit a CU");
};

// Units of 16 bytes (a group's 32 codes) of row r stand at u ^ swizzle, which
// spreads what the lanes of a read take over the banks.  K: one word each of
// 16 rows and 4 places.  V: half a unit each of rows 4 i .. 4 i + 3 and 16 on
// for two i at a time.  96 channels: 48-byte rows, spread as they are.
template <int G>
__device__ __forceinline__ int k_place(int r, int u) {
  return G == 2 ? u ^ ((r >> 3) & 1) : G == 4 ? u ^ ((r >> 2) & 3) : G == 8 ? u ^ ((r >> 1) & 7) : u;
}
template <int G>
__device__ __forceinline__ int v_place(int r, int u) {
  return G == 2   ? u ^ ((r >> 4) & 1)
         : G == 4 ? u ^ (((r >> 2) & 1) | ((r >> 3) & 2))
         : G == 8 ? u ^ (((r >> 1) & 3) | ((r >> 2) & 4))
                  : u;
}

// Eight codes as an operand: codes 0, 4, 1, 5, 2, 6, 3, 7 of the word, times
// 2^-24, the second and fourth pair times 2^-20.
__device__ __forceinline__ f16x8 operand(uint32_t w) {
  u32x4 r;
  r[0] = w & 0x000f000fu;
  r[1] = w & 0x00f000f0u;
  w >>= 8;
  r[2] = w & 0x000f000fu;
  r[3] = w & 0x00f000f0u;
  return __builtin_bit_cast(f16x8, r);
}
// The same less 8, times 2^-9 all of them, as normal numbers: one exact
// fused multiply-add per pair.
__device__ __forceinline__ f16x8 centred_operand(uint32_t w) {
  const f16_t even = (f16_t)0x1p15f, odd = (f16_t)0x1p11f, eight = (f16_t)0x1p-6f;
  return __builtin_elementwise_fma(operand(w), (f16x8){even, even, odd, odd, even, even, odd, odd},
                                   (f16x8){-eight, -eight, -eight, -eight, -eight, -eight, -eight, -eight});
}
constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};

// gfx950 transposing read of 4-bit elements: lane k of 16 points at 16 of
// them; lane j receives element j of all 16, lane k's as nibble k.
__device__ __forceinline__ u32x2 lds_read_tr4x16(const char* p) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
      (__attribute__((address_space(3))) i32x2*)(p));
  return __builtin_bit_cast(u32x2, v);
}

// (by value: a bit cast of a vector's element in place reads its element 0)
__device__ __forceinline__ f16x2 halves(uint32_t x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ uint32_t pair(f16_t x, f16_t y) {
  return __builtin_bit_cast(uint32_t, (f16x2){x, y});
}
__device__ __forceinline__ u16x2 bits16(uint32_t x) { return __builtin_bit_cast(u16x2, x); }

__device__ __forceinline__ f16x8 four(const f16x2* x) {
  return (f16x8){x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

// (left to itself the compiler first makes every operand canonical)
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// The sum over the R columns of one query.
template <int R>
__device__ __forceinline__ float over_slots(float x) {
  auto turned = [](float y, auto ctrl) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y), decltype(ctrl)::value,
                                                      0xf, 0xf, true));
  };
  x += turned(x, Par<0x128>{});                          // by 8 columns of 16
  if constexpr (R == 4) x += turned(x, Par<0x124>{});  // and 4
  return x;
}

// The largest (and the sum) over the four lanes of a column.
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

__device__ __forceinline__ float column_weight(float m, float M) { return fast_exp2(m - M); }

template <typename TO>
__device__ __forceinline__ void store4(TO* p, f32x4 x, bool vec) {
  typedef TO TO4 __attribute__((ext_vector_type(4)));
  const TO4 y = {from_f32<TO>(x[0]), from_f32<TO>(x[1]), from_f32<TO>(x[2]), from_f32<TO>(x[3])};
  if (vec) {
    *(TO4*)p = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = y[i];
  }
}

// Channels c .. c + 3 of a row of the output: O / l, gated; zeros where the
// token has no row.
template <typename T>
__device__ __forceinline__ void write_out(const Q4Args& a, int64_t at, f32x4 o, float l, bool live) {
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = l == 0.f ? __builtin_nanf("") : o[i] * inv;
    if (a.gate != nullptr) {
      const T* g = (const T*)a.gate + at;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= fast_sigmoid(to_f32(g[i]));
    }
  }
  switch (a.out_dtype) {
    case ALPX_F32: store4((float*)a.out + at, y, a.vec); break;
    case ALPX_F16: store4((f16_t*)a.out + at, y, a.vec); break;
    default: store4((bf16_t*)a.out + at, y, a.vec);
  }
}

// One block per (share of the rows, kv head, column tile): a column is one
// query head of one token.  Each wave runs alone over its own tiles, with its
// own ring in LDS, up to the end of a sequence, where the four meet.
// Alone (no `found`): a share is a whole sequence, and there is nothing to join.
//
// Few columns are bound by memory on long contexts: 4 x 1 on 131072 rows, 32/8
// heads of 128, fp16, 672 MB in 140 us (4.8 TB/s; the loads alone, without the
// arithmetic, 5.2).  On shorter ones the start and the end count, some 6 us:
// the shares, pages, queries and first tiles of a block, and its waves' meeting
// (16 x 1 ragged 8192, 95 MB: 25 to 28 us and 4 for the join).  Many columns are bound
// by the vector unit, which multiplies by steps, takes P apart and forms
// operands (4 x 64 on 4133 rows: busy 59% of the time, the matrix unit 22%).
template <typename S>
__global__ void __launch_bounds__(64 * kWaves, S::kPerCu) q4_kernel(Q4Args a) {
  typedef typename S::T T;
  constexpr int G = S::G, CT = S::CT, CP = S::CP, R = S::R, NT = S::NT, TP = S::TP, QP = S::QP, D = S::D, RING = S::RING;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // The column tiles of one (slot, kv head) run next to each other on one
  // XCD, whose L2 then holds the tiles that they all read.
  const int xcd = blockIdx.x % kXcds, place = blockIdx.x / kXcds;
  const int ct = place % a.col_tiles;
  const int unit = (place / a.col_tiles) * kXcds + xcd;
  const int kvh = unit / a.slots, slot = unit % a.slots;
  if (kvh >= a.kv_heads) return;
  const bool alone = a.found == nullptr;
  Share sh;
  if (alone) {
    sh = {};
    sh.b = slot;
    uniform_rows(a, slot, sh.P, sh.end);
    sh.tiles = sh.nt = (sh.end + S::kStepRows - 1) / S::kStepRows;
  } else {
    sh = find_share<S::kStepRows>(a, slot, unit == 0 && ct == 0 && wave == 0);
    if (sh.b < 0) return;  // fewer tiles than slots
  }

  // This lane's parts of a tile's loads: 16 bytes of codes, row L / G, and of
  // scales, plane L / 4.
  uint32_t kofs[S::kCodeLoads], vofs[S::kCodeLoads];
#pragma unroll
  for (int n = 0; n < S::kCodeLoads; ++n) {
    const int L = 64 * n + lane, r = L / G, u = L % G;
    kofs[n] = (uint32_t)(16 * (r * G + k_place<G>(r, u)));
    vofs[n] = (uint32_t)(16 * (r * G + v_place<G>(r, u)));
  }
  const uint32_t sofs = ((uint32_t)(lane >> 2) << (a.page_shift + 1)) + 16u * (lane & 3);
  const uint32_t plane_span = ((uint32_t)(2 * G - 1) << (a.page_shift + 1)) + 64u;
  char* const ring = smem + wave * (RING * S::kStepB);
  const uint32_t lring =
      (uint32_t)(uintptr_t)(lds_void_t*)smem + (uint32_t)(wave * (RING * S::kStepB));

  for (;;) {
    const int b = sh.b, P = sh.P, end = sh.end, nt = sh.nt;
    if (!alone && sh.t0 == 0 && kvh == 0 && ct == 0 && tid == 0)
      a.found[b] = make_int4(slot, sh.s1, P, end);
    const int32_t* table = a.table + (int64_t)b * a.max_pages;
    const int first = sh.t0 + wave;                        // this wave's steps
    // (none where no column of the block has a token)
    const bool any = P + ct * S::kCols / a.group < end;
    const int mine = any ? (nt - wave + kWaves - 1) / kWaves : 0;
    const int last_row = max(end - 1, 0);
    auto row_of = [&](int i, int u) __attribute__((always_inline)) {
      return min((first + kWaves * i) * S::kStepRows + u * kRows, last_row & -kRows);
    };
    struct Pages {
      int p[TP];
    };
    auto pages_of = [&](int i) __attribute__((always_inline)) {
      Pages r;
#pragma unroll
      for (int u = 0; u < TP; ++u) r.p[u] = load_const(table + (row_of(i, u) >> a.page_shift));
      return r;
    };
    // (the nontemporal hint on codes that no other block reads: 4 x 1 on 131072
    // rows, 32/8 heads of 128, 150 -> 140 us; on the scales too, the same)
    auto load = [](i32x4 r, uint32_t lds, uint32_t ofs) __attribute__((always_inline)) {
      if constexpr (S::kOnce) lds_dma16_once(r, lds, ofs);
      else lds_dma16(r, lds, ofs);
    };
    // Asks for step i of this wave; tiles behind the last row bring the last one.
    auto load_step = [&](int i, Pages pages, int stage) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        const int page = min(max(pages.p[u], 0), a.num_pages - 1);
        const int row = row_of(i, u) & ((1 << a.page_shift) - 1);
        const uint64_t head = (uint64_t)((int64_t)page * a.kv_heads + kvh);
        const uint64_t cofs = ((head << a.page_shift) + row) * (16 * G);
        const uint64_t pofs = ((head * (2 * G) << a.page_shift) + row) * 2;
        const uint32_t to = lring + stage * S::kStepB + u * S::kTileB;
        const i32x4 rk = rsrc_words((uint64_t)(uintptr_t)a.kc + cofs, S::kCodeB);
        const i32x4 rv = rsrc_words((uint64_t)(uintptr_t)a.vc + cofs, S::kCodeB);
        const i32x4 sk = rsrc_words((uint64_t)(uintptr_t)a.ks + pofs, plane_span);
        const i32x4 sv = rsrc_words((uint64_t)(uintptr_t)a.vs + pofs, plane_span);
        constexpr int kPart = S::kCodeB / 16 % 64;  // lanes of a last, partial load
#pragma unroll
        for (int n = 0; n < S::kCodeLoads; ++n)
          if (kPart == 0 || n + 1 < S::kCodeLoads || lane < kPart)
            load(rk, to + n * 1024, kofs[n]);
        if (8 * G == 64 || lane < 8 * G) lds_dma16(sk, to + 2 * S::kCodeB, sofs);
#pragma unroll
        for (int n = 0; n < S::kCodeLoads; ++n)
          if (kPart == 0 || n + 1 < S::kCodeLoads || lane < kPart)
            load(rv, to + S::kCodeB + n * 1024, vofs[n]);
        if (8 * G == 64 || lane < 8 * G) lds_dma16(sv, to + 2 * S::kCodeB + S::kScaleB, sofs);
      }
    };
    const int slot_of = hl / CP;  // packed: which of R groups the column stands for
    // This lane's octet of every group of its column's row of q: asked for
    // before the tiles, behind which it would arrive.
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 raw[CT][G];
    int lim[CT];        // rows that the column sees; 0: it has none
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int col = ct * S::kCols + 16 * c + hl % CP;
      const int node = col / a.group;
      const bool live = node < a.nodes && P + node < end;
      lim[c] = live ? P + node + 1 : 0;
      const int64_t row =
          ((int64_t)b * a.nodes + (live ? node : 0)) * a.q_heads + kvh * a.group +
          (live ? col - node * a.group : 0);
      const T* qp = (const T*)a.q + row * D + 8 * quad;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (a.vec) {
          raw[c][g] = *(const T8*)(qp + 32 * g);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) raw[c][g][e] = qp[32 * g + e];
        }
      }
    }
    Pages pages[RING];
#pragma unroll
    for (int i = 0; i < RING; ++i)
      if (i < mine) pages[i] = pages_of(i);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int g = 0; g < G; ++g) asm volatile("" : "+v"(raw[c][g]));  // (they are here)
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
      if (i < mine) load_step(i, pages[i], i);
    Pages next_pages = pages[RING - 1];

    // The queries, as operands: scaled by a power of two to a largest value
    // below 2^15.
    f16x8 q[CT][QP][G];
    f16x8 qsum[CT];     // sums over groups, in parts: groups `quad` (and quad + 4)
    float own_sum[NT];  // packed: of this column's groups
    float k1[CT];       // what a score is to be multiplied by
    float m[CT];
    uint32_t nans[CT];  // groups that a row of this column made NaN
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      m[c] = -3.0e38f;
      nans[c] = 0;
      float x[G][8];
      float most = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[g][e] = to_f32((T)raw[c][g][e]);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[g][e]));
      }
      most = column_max(most);
      int ex = 0;
      if (most > 0.f && most < __builtin_inff()) ex = 14 - max(__builtin_amdgcn_frexp_expf(most) - 1, -90);
      const float f = ldexpf(1.f, ex);
      // (never 0: a masked score, -inf, has to stay one)
      k1[c] = fmaxf(ldexpf(a.scale_log2, (S::kCentred ? 9 : 24) - ex), 0x1p-126f);
      u32x4 sums = {0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = x[g][kOrder[e]] * f;
          const float z = !S::kCentred && (e & 2) ? y * 0.0625f : y;
          const f16_t hi = (f16_t)z;
          const bool mine = !S::kPacked || g % R == slot_of;  // this column's group
          q[c][0][g][e] = mine ? hi : (f16_t)0.f;
          float z1 = (float)hi;  // what the products take
          if constexpr (QP == 2) {
            const f16_t lo = (f16_t)(z - z1);
            q[c][1][g][e] = mine ? lo : (f16_t)0.f;
            z1 += (float)lo;
          }
          s += !S::kCentred && (e & 2) ? z1 * 16.f : z1;
        }
        if constexpr (S::kPacked) {
          s = column_sum(s);
          if (g % R == 0) own_sum[g / R] = 0.f;
          if (g % R == slot_of) own_sum[g / R] = s * S::kSumUnit;
          continue;
        }
        // the group's sum in units that keep it below 2^14: in three parts, or,
        // where steps take 8 times it, both in two (22 bits, as q)
        s = column_sum(s) * S::kSumScale;
        const f16_t p0 = (f16_t)s, p1 = (f16_t)(s - (float)p0);
        uint32_t rest;
        if constexpr (S::kCentred) rest = pair(p0 * (f16_t)8.f, p1 * (f16_t)8.f);
        else rest = pair((f16_t)(s - (float)p0 - (float)p1), (f16_t)0.f);
        if ((g & 3) == quad) {
          sums[g / 4 * 2] = pair(p0, p1);
          sums[g / 4 * 2 + 1] = rest;
        }
      }
      qsum[c] = __builtin_bit_cast(f16x8, sums);
    }

    f32x4 o[CT][2 * G];  // O^T[channel 16 n + 4 quad + r][column] of the codes less 8
    float om[CT][S::kBases];  // sums of p (m + 8 d) of groups `quad` (and quad + 4)
    float l[CT];              // the sum of p (G = 8: of this lane's keys)
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      l[c] = 0.f;
#pragma unroll
      for (int h = 0; h < S::kBases; ++h) om[c][h] = 0.f;
#pragma unroll
      for (int n = 0; n < 2 * G; ++n) o[c][n] = (f32x4)(0.f);
    }
    // byte offsets of this lane's operands in a tile
    int kadr[G], vadr[G];
    const int vk = lane & 7;  // nibbles 0, 4 / 1, 5 / 2, 6 / 3, 7: keys 4 quad + 0 .. 3, and 16 on
    const int vrow = 4 * quad + ((vk & 1) << 1) + (vk >> 2) + ((vk & 2) << 3);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      kadr[g] = hl * 16 * G + 16 * k_place<G>(hl, g) + 4 * quad;  // (row hl + 16: the same place)
      vadr[g] = S::kCodeB + vrow * 16 * G + 16 * v_place<G>(vrow, g) + 8 * ((lane >> 3) & 1);
    }
    const bool has_m = quad < G;
    const int mk = (has_m ? quad : 0) * 64 + 2 * hl;  // steps of K; least values from plane G on
    // and of V: rows of an operand, whose results a lane of the group's quad gets
    // next to each other: least values, steps less than 0, ones (G = 8: those of
    // group quad, then of quad + 4; the sum of p without the matrix unit)
    const int vg = G == 8 ? (hl >> 2) + 4 * ((hl >> 1) & 1) : min(hl >> 2, G - 1);
    const int mv = (((G == 8 ? hl & 1 : hl & 3) == 0 ? G : 0) + vg) * 64 + 8 * quad;
    const uint32_t sign = hl & 1 ? 0x80008000u : 0u;  // of steps
    const bool ones = G < 8 && (hl & 3) >= 2;
    // steps of four keys; packed: of this column's group of the first R (unused
    // columns take the last group's, for sums of zeros)
    const int dadr = 8 * quad + (S::kPacked ? 64 * min(slot_of, G - 1) : 0);
    const int dlast = 8 * quad + 64 * min((NT - 1) * R + slot_of, G - 1);  // of the last R

    // Step i, which lies in stage `stage` of the ring (a constant: offsets in
    // the ring are then part of the LDS instructions).
    auto step = [&](auto stage_, int i) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_)::value;
      // (the reads of the step before, whose stage this fills, are done)
      wait_tiles<63>();
      if (i + RING - 1 < mine) {
        load_step(i + RING - 1, next_pages, (stage + RING - 1) % RING);
        next_pages = pages_of(min(i + RING, mine - 1));
      }
      const int left = mine - 1 - i;
      if (left >= RING - 1) wait_tiles<(RING - 1) * S::kStepLoads>();
      else if (RING > 3 && left == 2) wait_tiles<2 * S::kStepLoads>();
      else if (RING > 2 && left == 1) wait_tiles<S::kStepLoads>();
      else wait_tiles<0>();
      char* const tiles = ring + stage * S::kStepB;
      const int key0 = (first + kWaves * i) * S::kStepRows;
      const bool tail = key0 + S::kStepRows > P + 1;  // some column does not see all of it
      if (tail) {
        // rows past the last: their scales count as zeros; rows that some
        // columns do not see and that are not finite: set apart
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          uint16_t* s = (uint16_t*)(tiles + u * S::kTileB + 2 * S::kCodeB + S::kScaleB);
          const int rows = end - key0 - kRows * u;
          bool odd = false;
          for (int x = lane; x < 2 * G * kRows; x += 64) {
            if ((x & (kRows - 1)) >= rows) s[x] = 0;
            odd |= (s[x] & 0x7fff) >= 0x7c00;
          }
          if (__ballot(odd) != 0) {
            for (int r = 0; r < kRows && r < rows; ++r) {
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const int sd = s[g * kRows + r] & 0x7fff, sm = s[(G + g) * kRows + r] & 0x7fff;
                if (sd < 0x7c00 && sm < 0x7c00) continue;
#pragma unroll
                for (int c = 0; c < CT; ++c)
                  if (key0 + kRows * u + r < lim[c]) nans[c] |= 1u << g;
                s[g * kRows + r] = 0;
                s[(G + g) * kRows + r] = 0;
              }
            }
          }
        }
        asm volatile("" ::: "memory");
      }

      // S^T: key 32 u + 16 kt + 4 quad + r of the step is value 8 u + 4 kt + r
      float s[CT][8 * TP];
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        const char* const tile = tiles + u * S::kTileB;
        const char* const sc_k = tile + 2 * S::kCodeB;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          if constexpr (S::kPacked) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int g = R * t; g < min(R * t + R, G); ++g) {
                const uint32_t w = *(const uint32_t*)(tile + kadr[g] + 256 * G * kt);
                const f16x8 kx = S::kCentred ? centred_operand(w) : operand(w);
                if constexpr (QP == 2) x = mfma16x16x32(kx, q[0][1][g], x);
                x = mfma16x16x32(kx, q[0][0][g], x);
              }
              const char* const dp = sc_k + (t + 1 < NT ? dadr + 64 * R * t : dlast) + 32 * kt;
              const f16x4 d = *(const f16x4*)dp, least = *(const f16x4*)(dp + 64 * G);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float& y = s[0][8 * u + 4 * kt + r];
                const float base = S::kCentred ? fmaf((float)d[r], 8.f, (float)least[r]) : (float)least[r];
                y = fmaf(base, own_sum[t], t == 0 ? 0.f : y);
                y = fmaf((float)d[r], x[r], y);
              }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[0][8 * u + 4 * kt + r] = over_slots<R>(s[0][8 * u + 4 * kt + r]);
            continue;
          }
          // least values of this lane's groups against the parts of the sums,
          // steps against 8 times these
          f16x8 mf = {};
#pragma unroll
          for (int h = 0; h < (G + 3) / 4; ++h) {
            const char* mp = sc_k + mk + 4 * h * 64 + 32 * kt;
            f16_t least = *(const f16_t*)(mp + G * 64), d = least;
            if constexpr (S::kCentred) d = *(const f16_t*)mp;
            if (G % 4 != 0 && !has_m) least = d = (f16_t)0.f;
            mf[4 * h] = mf[4 * h + 1] = least;
            mf[4 * h + 2] = mf[4 * h + 3] = d;
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const f32x4 x = mfma16x16x32(mf, qsum[c], (f32x4)(0.f));
#pragma unroll
            for (int r = 0; r < 4; ++r) s[c][8 * u + 4 * kt + r] = x[r] * S::kSumUnit;
          }
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const uint32_t w = *(const uint32_t*)(tile + kadr[g] + 256 * G * kt);
            const f16x8 kx = S::kCentred ? centred_operand(w) : operand(w);
            const f16x4 d = *(const f16x4*)(sc_k + dadr + 64 * g + 32 * kt);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              f32x4 x = {0.f, 0.f, 0.f, 0.f};
              if constexpr (QP == 2) x = mfma16x16x32(kx, q[c][1][g], x);
              x = mfma16x16x32(kx, q[c][0][g], x);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float& y = s[c][8 * u + 4 * kt + r];
                y = fmaf((float)d[r], x[r], y);
              }
            }
          }
        }
      }
      if (tail) {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int e = 0; e < 8 * TP; ++e)
            if (key0 + 32 * (e >> 3) + 16 * (e >> 2 & 1) + 4 * quad + (e & 3) >= lim[c])
              s[c][e] = -__builtin_inff();
      }

      // The reference of the probabilities: the largest score so far, less
      // kSlack, and as much more as V's steps pass 1, so that p d stays in
      // float16.
      float lift = 0.f;
      {
        u16x2 y = {0, 0};
        u32x4 x[TP];
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          x[u] = *(const u32x4*)(tiles + u * S::kTileB + 2 * S::kCodeB + S::kScaleB +
                                 16 * (lane < 4 * G ? lane : 0));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y = __builtin_elementwise_max(y, bits16(x[u][e]));
        }
        y = __builtin_elementwise_sub_sat(y, (u16x2){0x3c00, 0x3c00});
        if (__ballot(__builtin_bit_cast(uint32_t, y) != 0) != 0) {
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < 4 * TP; ++e) {
            const f16x2 h = halves(x[e / 4][e % 4]);
            most = fmaxf(most, fmaxf(fabsf((float)h[0]), fabsf((float)h[1])));
          }
#pragma unroll
          for (int off = 1; off < 64; off <<= 1) most = fmaxf(most, __shfl_xor(most, off));
          lift = fminf(fmaxf((float)__builtin_amdgcn_frexp_expf(most), 0.f), 16.f);
        }
      }
      float top[CT];
      bool over = false;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        float x = max3(s[c][0], s[c][1], s[c][2]);
#pragma unroll
        for (int e = 3; e + 1 < 8 * TP; e += 2) x = max3(x, s[c][e], s[c][e + 1]);
        x = max3(x, s[c][8 * TP - 1], x);
        top[c] = fmaf(x, k1[c], lift);
        over |= top[c] > m[c] + kSlack;
      }
      if (__ballot(over) != 0) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          // (a whole number: the lift and the weight of what was are exact)
          const float M = ceilf(fmaxf(m[c], column_max(top[c])));
          const float w = column_weight(m[c], M);
          m[c] = M;
          l[c] *= w;
#pragma unroll
          for (int h = 0; h < S::kBases; ++h) om[c][h] *= w;
#pragma unroll
          for (int n = 0; n < 2 * G; ++n) o[c][n] *= w;
        }
      }

      // P in two parts of float16
      f16x2 ph[CT][4 * TP], pl[CT][4 * TP];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const float base = kLift - m[c];
#pragma unroll
        for (int e = 0; e < 4 * TP; ++e) {
          const float x0 = fast_exp2(fmaf(s[c][2 * e], k1[c], base));
          const float x1 = fast_exp2(fmaf(s[c][2 * e + 1], k1[c], base));
          if constexpr (G == 8) l[c] += x0 + x1;
          ph[c][e] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
          pl[c][e] = (f16x2){(f16_t)(x0 - (float)ph[c][e][0]), (f16_t)(x1 - (float)ph[c][e][1])};
        }
      }
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        // Least values and 8 steps, as exact as they stand, and joined tile by
        // tile: their sums over all rows would grow past what they leave.  The
        // unit rounds its sums downwards, small ones first the least (float32, 500
        // rows: 5e-7 of the result, large first 7e-7); of least values and negated
        // steps, mostly of one sign, what it takes cancels (131072 rows: 6e-7; with
        // steps as they are 1.8e-6).
        const char* mp = tiles + u * S::kTileB + 2 * S::kCodeB + S::kScaleB + mv;
        const u32x2 m0 = *(const u32x2*)mp, m1 = *(const u32x2*)(mp + 32);
        constexpr uint32_t kOnes = 0x3c003c00u;
        const f16x8 mf = __builtin_bit_cast(
            f16x8, (u32x4){ones ? kOnes : m0[0] ^ sign, ones ? kOnes : m0[1] ^ sign,
                           ones ? kOnes : m1[0] ^ sign, ones ? kOnes : m1[1] ^ sign});
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          f32x4 x = mfma16x16x32(mf, four(pl[c] + 4 * u), (f32x4)(0.f));
          x = mfma16x16x32(mf, four(ph[c] + 4 * u), x);
          om[c][0] += fmaf(x[1], -8.f, x[0]);
          if constexpr (G == 8) om[c][S::kBases - 1] += fmaf(x[3], -8.f, x[2]);
          else l[c] += x[2];
        }
      }
      // P times the steps at dp of tile u, in two parts
      f16x2 hi[CT][TP][4], lo[CT][TP][4];
      auto weigh = [&](const char* dp, int u) __attribute__((always_inline)) {
        const u32x2 d01 = *(const u32x2*)dp, d23 = *(const u32x2*)(dp + 32);
        const f16x2 d[4] = {halves(d01[0]), halves(d01[1]), halves(d23[0]), halves(d23[1])};
#pragma unroll
        for (int c = 0; c < CT; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f16x2 p = ph[c][4 * u + e];
            const f16x2 h = p * d[e];
            hi[c][u][e] = h;
            // what the rounding took, and the second part's share
            lo[c][u][e] = __builtin_elementwise_fma(pl[c][4 * u + e], d[e],
                                                    __builtin_elementwise_fma(p, d[e], -h));
          }
        }
      };
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          const char* const tile = tiles + u * S::kTileB;
          const u32x2 w = lds_read_tr4x16(tile + vadr[g]);
          const f16x8 v0 = centred_operand(w[0]), v1 = centred_operand(w[1]);
          if (!S::kPacked || g % R == 0) {  // the groups of one accumulator share their P d
            const char* const dp = tile + 2 * S::kCodeB + S::kScaleB +
                                   (!S::kPacked || g / R + 1 < NT ? dadr + 64 * g : dlast);
            weigh(dp, u);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            o[c][2 * g] = mfma16x16x32(v0, four(hi[c][u]), o[c][2 * g]);
            o[c][2 * g + 1] = mfma16x16x32(v1, four(hi[c][u]), o[c][2 * g + 1]);
            o[c][2 * g] = mfma16x16x32(v0, four(lo[c][u]), o[c][2 * g]);
            o[c][2 * g + 1] = mfma16x16x32(v1, four(lo[c][u]), o[c][2 * g + 1]);
          }
        }
      }
    };
    for (int i = 0; i < mine; i += RING)
      static_for<0, RING>([&](auto j) {
        if (i + decltype(j)::value < mine) step(j, i + decltype(j)::value);
      });

    // The waves meet: each leaves its reference, its sum and O, with the
    // least values' part in it.
    __syncthreads();  // nobody reads tiles any more
    f32x4* const st = (f32x4*)(smem + kWaves * 16 * S::kMergeRow * 4);
    const bool whole = alone || nt == sh.tiles;
    const int64_t seg = (((int64_t)(slot + b) * a.kv_heads + kvh) * a.col_tiles + ct) * S::kCols;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float* const mo = (float*)smem + (wave * 16 + hl % CP) * S::kMergeRow;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float pm = __shfl(om[c][g >> 2], (g & 3) * 16 + hl);
        const float bad = (nans[c] >> g & 1) ? __builtin_nanf("") : 0.f;
#pragma unroll
        for (int n = 2 * g; n < 2 * g + 2; ++n) {
          f32x4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = fmaf(o[c][n][r], kUnit, pm) + bad;
          if (!S::kPacked || g % R == slot_of) *(f32x4*)(mo + 16 * n + 4 * quad) = x;
        }
      }
      const float sum_p = G == 8 ? column_sum(l[c]) : l[c];
      if (lane < CP) st[(wave * CT + c) * 16 + hl] = (f32x4){m[c], sum_p, 0.f, 0.f};
      __syncthreads();
      for (int x = tid; x < CP * 8 * G; x += 64 * kWaves) {
        const int cl = x / (8 * G), ch = 4 * (x - cl * (8 * G));
        const int col = ct * S::kCols + 16 * c + cl, node = col / a.group;
        if (node >= a.nodes) continue;
        float M = -3.0e38f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, st[(w * CT + c) * 16 + cl][0]);
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const f32x4 v = st[(w * CT + c) * 16 + cl];
          const float wt = column_weight(v[0], M);
          sum = fmaf(v[1], wt, sum);
          y += *(const f32x4*)((float*)smem + (w * 16 + cl) * S::kMergeRow + ch) * wt;
        }
        if (whole) {
          const int64_t row = ((int64_t)b * a.nodes + node) * a.q_heads + kvh * a.group +
                              (col - node * a.group);
          write_out<T>(a, row * D + ch, y, sum, P + node < end);
        } else if (P + node < end) {
          *(f32x4*)(a.part_o + (seg + 16 * c + cl) * D + ch) = y;
          if (ch == 0) a.part_st[seg + 16 * c + cl] = make_float2(M, sum);
        }
      }
      // the space goes to the next columns, or tiles
      if (c + 1 < CT || sh.left != 0) __syncthreads();
    }
    if (sh.left == 0) return;
    // the next sequence that has rows
    do {
      ++sh.b;
      uniform_rows(a, sh.b, sh.P, sh.end);
      sh.tiles = (sh.end + S::kStepRows - 1) / S::kStepRows;
    } while (sh.tiles == 0);
    sh.t0 = 0;
    sh.nt = min(sh.left, sh.tiles);
    sh.left -= sh.nt;
    sh.s1 = slot + (sh.tiles - sh.nt + sh.per - 1) / sh.per;
  }
}

// Joins the segments of the sequences that more than one slot has tiles of,
// and writes zeros for those without a row.  One block per COLS columns:
// 8 / COLS threads per channel quad take the segments in turn and meet in
// LDS.  One column a block where a sequence has many segments (4 x 1 on 32768
// rows, 32 segments of 256 channels: 4.0 us, four columns 9.5), four where
// there are many columns (4 x 64 on 4133 rows, 8192 of them: 6.5 us, one 8.9).
template <typename T, int G, int COLS>
__global__ void __launch_bounds__(64 * G) q4_join(Q4Args a, int cols, int tile_cols) {
  constexpr int D = 32 * G, kItems = 8 * G, kFlight = 4, kJoinShare = 8 / COLS;
  __shared__ f32x4 part[kJoinShare][COLS * kItems];
  __shared__ float2 st[kJoinShare][COLS];
  const int groups = (cols + COLS - 1) / COLS;
  const int cl = threadIdx.x / kItems % COLS;
  const int col = blockIdx.x % groups * COLS + cl, node = col / a.group;
  const int kvh = blockIdx.x / groups % a.kv_heads, b = blockIdx.x / groups / a.kv_heads;
  const int32_t* found = (const int32_t*)(a.found + b);
  const int s0 = load_const(found), s1 = load_const(found + 1);
  const int P = load_const(found + 2), end = load_const(found + 3);
  if (s0 == s1) return;  // written by its slot
  const int item = threadIdx.x % (COLS * kItems), w = threadIdx.x / (COLS * kItems);
  const int ch = 4 * (threadIdx.x % kItems);
  const bool live = node < a.nodes && P + node < end;
  float m = -3.0e38f, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const int ct = col / tile_cols;
    auto at = [&](int s) __attribute__((always_inline)) {
      return (((int64_t)(s + b) * a.kv_heads + kvh) * a.col_tiles + ct) * tile_cols +
             (col - ct * tile_cols);
    };
    for (int s = s0 + w; s <= s1; s += kJoinShare * kFlight) {
      float2 v[kFlight];
      f32x4 x[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int64_t row = at(min(s + kJoinShare * u, s1));  // past the last: again, unused
        v[u] = a.part_st[row];
        x[u] = *(const f32x4*)(a.part_o + row * D + ch);
      }
      float M = m;
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        if (s + kJoinShare * u <= s1) M = fmaxf(M, v[u].x);
      const float c = column_weight(m, M);
      l *= c;
      o *= c;
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        if (s + kJoinShare * u > s1) continue;
        const float cu = column_weight(v[u].x, M);
        l = fmaf(v[u].y, cu, l);
        o += x[u] * cu;
      }
      m = M;
    }
  }
  part[w][item] = o;
  if (ch == 0) st[w][cl] = make_float2(m, l);
  __syncthreads();
  if (w != 0 || node >= a.nodes) return;
  float M = -3.0e38f, sum = 0.f;
#pragma unroll
  for (int v = 0; v < kJoinShare; ++v) M = fmaxf(M, st[v][cl].x);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < kJoinShare; ++v) {
    const float c = column_weight(st[v][cl].x, M);
    sum = fmaf(st[v][cl].y, c, sum);
    y += part[v][item] * c;
  }
  const int64_t row =
      ((int64_t)b * a.nodes + node) * a.q_heads + kvh * a.group + (col - node * a.group);
  write_out<T>(a, row * D + ch, y, sum, live);
}

template <typename S>
Q4Kernel make() {
  return {(const void*)q4_kernel<S>, (const void*)q4_join<typename S::T, S::G, S::CT == 1 ? 1 : 4>,
          S::CT == 1 ? 1 : 4, S::kCols, S::kStepRows, S::kPerCu};
}

// Up to 16 columns one column tile, two tiles of 32 rows to a step where two
// blocks of them fit a CU (4 x 1 on 32768 rows of 256, one: two do not); up to
// 8 and 4 of them as queries times groups (16 x 1 ragged 8192, 4 queries a head:
// 31.2 us, 16 plain columns 34.9).  Of more, two column tiles to a block: K's and
// V's operands serve both (4 x 64 on 4133 rows: 61 us; four, which leave a wave
// a SIMD, 68; one 69).  Rings of three and four steps for one column tile take
// as long as two.  float32 queries of 128 channels keep 4 registers a lane of
// theirs in scratch (4 x 64 on 4133 rows: 69 us).
template <typename T>
Q4Kernel pick(int head_dim, int cols) {
  const int few = cols <= 4 ? 4 : cols <= 8 ? 8 : cols <= 16 ? 16 : 0;
  switch (head_dim) {
    case 64:
      return few == 0    ? make<Q4Shape<T, 2, 2, 16, 1, 4, 2>>()
             : few == 16 ? make<Q4Shape<T, 2, 1, 16, 2, 2, 3>>()
                         : make<Q4Shape<T, 2, 1, 8, 2, 2, 3>>();
    case 96:
      return few == 0    ? make<Q4Shape<T, 3, 2, 16, 1, 4, 2>>()
             : few == 16 ? make<Q4Shape<T, 3, 1, 16, 2, 2, 2>>()
             : few == 8  ? make<Q4Shape<T, 3, 1, 8, 2, 2, 2>>()
                         : make<Q4Shape<T, 3, 1, 4, 2, 2, 2>>();
    case 128:
      return few == 0    ? make<Q4Shape<T, 4, 2, 16, 1, 4, 2>>()
             : few == 16 ? make<Q4Shape<T, 4, 1, 16, 2, 2, 2>>()
             : few == 8  ? make<Q4Shape<T, 4, 1, 8, 2, 2, 2>>()
                         : make<Q4Shape<T, 4, 1, 4, 2, 2, 2>>();
    default:
      return few == 0    ? make<Q4Shape<T, 8, 2, 16, 1, 2, 1>>()
             : few == 16 ? make<Q4Shape<T, 8, 1, 16, 1, 2, 1>>()
             : few == 8  ? make<Q4Shape<T, 8, 1, 8, 1, 2, 1>>()
                         : make<Q4Shape<T, 8, 1, 4, 1, 2, 1>>();
  }
}

}  // namespace
}  // namespace alpx
