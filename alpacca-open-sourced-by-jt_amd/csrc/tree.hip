// Attention of a tree of drafted tokens over a K/V cache.
//
// Sequence b holds P_b rows that every draft sees (its prefix) and, behind
// them, one row for each of its n_b drafts.  Draft i sees the prefix and
// those rows P_b + j whose bit j is set in its mask (its ancestors and
// itself, in a tree):
//   out[b, i, h] = softmax_j(scale * q[b, i, h] . K[j, h / G]) . V[j, h / G]
// over the rows it sees, times sigmoid(gate) where given; a draft that sees
// no row, and drafts at or past n_b, give zeros, whatever their gate holds.
//
// The drafts of one sequence read the same rows, so a block takes columns =
// (draft, query head of one kv head) pairs, up to 128 of them, against one
// stream of K and V tiles: the cache is read once for all of them.  S^T =
// K Q^T and O^T = V^T P^T on MFMA tiles of 16 or 32 columns: a lane owns one
// column, keys lie in its registers, so its mask is one word per 32 keys,
// the softmax needs one or two exchanges with the other lanes of the column,
// and P feeds the second product from the registers the first one wrote.
//
// Few columns are bound by the rows' way from memory (16 sequences of 16
// drafts on 8192 rows, 32/8 heads of 128, fp16: 78 us = 6.9 TB/s in the
// loop, 90 with both ends of the launch, 7 more for the join), many by the
// products and what they read from LDS (4 of 64 on 32768 rows, 16/2 heads of
// 256, bf16: 166 us with the join = 830 TFLOP/s from a graph; back to back,
// at the power limit, 170 to 178 and 10), short ones by latency (8 on 508
// rows, float32: 7.2 + 4.3 us).
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "alpx_common.h"
#include "prefill_run.h"
#include "timing.h"
#include "wave_scan.h"

namespace alpx {
namespace {

// lds_dma16 for bytes that no other block reads (the nontemporal hint).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved; the clobber is intended
__device__ __forceinline__ void lds_dma16_once(i32x4 r, uint32_t lds, uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
               :
               : "s"(lds), "v"(voff), "s"(r)
               : "memory", "m0");
#else
  (void)r;
  (void)lds;
  (void)voff;
#endif
}
#pragma clang diagnostic pop

struct TreeArgs {
  const void* q;      // [B, N, Hq, D]
  const void* k;
  const void* v;
  const void* gate;   // null, or [B, N, Hq, Dv]
  void* out;          // [B, N, Hq, Dv]
  const uint32_t* masks;  // [B or 1, N, words] 32-bit words
  const int32_t* prefix;  // device [B]
  const int32_t* counts;  // device [B] or null (every sequence has N drafts)
  int64_t mask_b;         // words between the masks of two sequences (0: shared)
  int64_t ks_pos, ks_b, ks_h, vs_pos, vs_b, vs_h;  // elements
  // Paged caches (pages != null): row j of sequence b is row j % page size
  // of page pages[b * max_pages + j / page size]; ks_b / vs_b are the page
  // strides.
  const int32_t* pages;
  int page_shift, max_pages, num_pages;
  int words;
  int length, batch, nodes, q_heads, kv_heads, group, key_dim, value_dim;
  int col_tiles;      // column tiles per (sequence, kv head)
  int slots;          // shares of the rows per (kv head, column tile)
  float* part_o;      // segments of O, [segment, kv head, column group][DP / 4][32] x 4
  float2* part_st;    // reference score and sum of P of their columns
  int4* found;        // [batch]: first and last slot of a sequence, P, end
  float scale_log2;
  int out_dtype;
  int vec_k, vec_q, vec_o;  // rows of K and of q may be read, of out written in vectors
  int direct;         // vec_o, value_dim = DP: a slot writes its whole sequences
};

// Loads that may come through the scalar cache: what they read is written
// by no block of the launch.
__device__ __forceinline__ int load_const(const int32_t* p) {
  return __builtin_amdgcn_readfirstlane(
      *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p);
}

// Rows of sequence b: its prefix [0, P), its drafts [P, end).  A sequence
// without drafts has none: nobody reads its prefix.
__device__ __forceinline__ void rows_from(const TreeArgs& a, int prefix, int count, int& P,
                                          int& end) {
  P = min(max(prefix, 0), a.length);
  end = min(P + min(max(count, 0), a.nodes), a.length);
  if (end == P) P = end = 0;
}
__device__ __forceinline__ void lane_rows(const TreeArgs& a, int b, int& P, int& end) {
  rows_from(a, a.prefix[b], a.counts != nullptr ? a.counts[b] : a.nodes, P, end);
}

// The same of one sequence for the whole wave, through the scalar cache.
__device__ __forceinline__ void uniform_rows(const TreeArgs& a, int b, int& P, int& end) {
  rows_from(a, load_const(a.prefix + b), a.counts != nullptr ? load_const(a.counts + b) : a.nodes,
            P, end);
  P = __builtin_amdgcn_readfirstlane(P);
  end = __builtin_amdgcn_readfirstlane(end);
}

// Shares of the rows: every slot gets a run of tiles of BK rows, cut on the
// device since only it knows the lengths.
//
// Where the sequences divide well, a run belongs to one of them: the shortest
// run length is searched with which all sequences' runs fit the slots, and
// each sequence is cut into equal runs.  Otherwise the sequences' tiles, one
// sequence after the other, are dealt out in runs of equal length, and a run
// may end one sequence and begin another, which costs it about kTurnOver
// tiles of waiting (for the next queries and first tiles).
//
// Slot s leaves the partial state of its tiles of sequence b in segment
// s + b: both rise along the runs, so no two segments share a number, and
// there are at most slots + batch.  A run that holds a whole sequence writes
// its output and leaves no partial state, only a mark whether that output is
// finite.
struct Share {
  int b;       // the sequence, -1: none
  int P, end;  // its rows: [0, P) the prefix, [P, end) the drafts
  int tiles;   // its tiles
  int t0, nt;  // the slot's: nt tiles of it from t0 on
  int left;    // and as many of the next sequences
  int s1;      // the last slot that has tiles of it
  int per;     // tiles per slot
};
constexpr int kTurnOver = 4;

__device__ __forceinline__ int div_up(int x, int y) {
  return (int)(((unsigned)x + (unsigned)y - 1u) / (unsigned)y);
}

// The first share of slot `slot`.  Every lane of a wave calls this, and gets
// the same.  `first_of_all`: sequences without a row are noted for the join (the
// others are by the slot that begins them).
template <int BK>
__device__ __forceinline__ Share find_share(const TreeArgs& a, int slot, bool first_of_all) {
  const int lane = threadIdx.x & 63;
  auto rows_of = [&](int b0, int& P, int& end) __attribute__((always_inline)) {
    P = end = 0;
    if (b0 + lane < a.batch) lane_rows(a, b0 + lane, P, end);
    return (end + BK - 1) / BK;
  };
  int P, end;
  int nt = rows_of(0, P, end);  // the first 64 sequences stay in registers
  int all = wave_total(nt);
  auto note_empty = [&](int b, int tiles) __attribute__((always_inline)) {
    if (first_of_all && tiles == 0 && b < a.batch) a.found[b] = make_int4(0, -1, 0, 0);
  };
  note_empty(lane, nt);
  for (int b0 = 64; b0 < a.batch; b0 += 64) {
    int p, e;
    const int n = rows_of(b0, p, e);
    all += wave_total(n);
    note_empty(b0 + lane, n);
  }
  const int per = max(1, div_up(all, a.slots));
  Share r = {};
  r.b = -1;
  int lo = per, hi = per;
  if (a.batch <= 64) {
    bool fits = wave_total(div_up(nt, per)) <= a.slots;
    if (!fits && a.slots > a.batch) {
      hi = min(div_up(all, a.slots - a.batch), per + kTurnOver + 1);
      while (hi - lo > 1) {  // lo does not fit, hi does or is too long
        const int mid = (lo + hi) >> 1;
        if (wave_total(div_up(nt, mid)) <= a.slots) hi = mid; else lo = mid;
      }
      fits = hi <= per + kTurnOver;
    }
    if (fits) {
      const int runs = div_up(nt, hi), before = wave_before(runs);
      const bool mine = slot >= before && slot < before + runs;
      const unsigned long long hit = __ballot(mine);
      if (hit == 0) return r;
      const int src = __ffsll((long long)hit) - 1;
      const int n = __builtin_amdgcn_readlane(runs, src);
      r.b = src;
      r.P = __builtin_amdgcn_readlane(P, src);
      r.end = __builtin_amdgcn_readlane(end, src);
      r.tiles = __builtin_amdgcn_readlane(nt, src);
      const int s0 = __builtin_amdgcn_readlane(before, src);
      r.s1 = s0 + n - 1;
      const int q = r.tiles / n, more = r.tiles - q * n, i = slot - s0;
      r.t0 = i * q + min(i, more);
      r.nt = q + (i < more ? 1 : 0);
      return r;
    }
  }
  const int want = slot * per;
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (b0 > 0) nt = rows_of(b0, P, end);
    const int first = base + wave_before(nt);
    const bool mine = want >= first && want < first + nt;
    const unsigned long long hit = __ballot(mine);
    if (hit != 0) {
      const int src = __ffsll((long long)hit) - 1;
      const int f = __builtin_amdgcn_readlane(first, src);
      r.b = b0 + src;
      r.P = __builtin_amdgcn_readlane(P, src);
      r.end = __builtin_amdgcn_readlane(end, src);
      r.tiles = __builtin_amdgcn_readlane(nt, src);
      r.s1 = (f + r.tiles - 1) / per;
      r.per = per;
      r.t0 = want - f;
      const int run = min(per, all - want);
      r.nt = min(run, r.tiles - r.t0);
      r.left = run - r.nt;
      return r;
    }
    base += __builtin_amdgcn_readlane(first + nt, 63) - base;
  }
  return r;
}

__device__ __forceinline__ f32x16 mfma32x32x16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32x32x16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32x32x2(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// fp16 probabilities are formed 2^kLift times as large as their reference
// says (the sums too, so it cancels): with kRescale they stay below 2^15, and
// weights down to 2^-21 of the largest, not 2^-14, keep all their bits.  Many
// rows of small weight beside a large one are what a first row that every
// draft attends to leaves.
template <typename T>
constexpr float kLift = std::is_same<T, f16_t>::value ? 7.f : 0.f;

// Shape of a kernel: T, DP (the head width rounded up to 64, 128 or 256), WC
// columns per wave (32, or 16 on the 16 x 16 MFMA), WQ waves side by side in
// columns, WK waves that share a column's keys, BK rows per K and V tile, a
// ring of RING tiles in LDS.
template <typename T_, int DP_, int WC_, int WQ_, int WK_, int BK_, int RING_>
struct Shape {
  typedef T_ T;
  static constexpr int DP = DP_, WC = WC_, WQ = WQ_, WK = WK_, BK = BK_, RING = RING_;
  static constexpr int NW = WQ * WK;             // waves
  static constexpr int kCols = WC * WQ;
  static constexpr int LPC = 64 / WC;            // lanes per column
  static constexpr int KG = BK / WK < 32 ? BK / WK : 32;  // keys of a wave at a time
  static constexpr int KR = BK / (KG * WK);      // such groups per tile
  static constexpr int NS = KG / LPC;            // scores per lane
  static constexpr int EPU = 16 / (int)sizeof(T);  // elements per 16-byte unit
  static constexpr int U = DP / EPU;             // units per row
  static constexpr int NQ = U / LPC;             // units of the query row per lane
  static constexpr int kRowB = DP * (int)sizeof(T);
  static constexpr int kTileB = BK * kRowB;
  static constexpr int kIW = kTileB / (1024 * NW);  // direct loads per wave and tile
  static constexpr int kTileLoads = 2 * kIW;     // the same for K and V
  static constexpr int NF = DP / (4 * LPC);      // 4-channel pieces of O^T per lane
  // The wide 16-bit kernels run the products of two tiles beside the softmax
  // of a third (see the loop).
  static constexpr bool kPipe = WC == 32 && sizeof(T) == 2 && RING == 2;
  // The narrow kernels have one column tile: nobody reads a tile twice.
  // (The hint on K and V / on V / on neither, 16 x 16 drafts on 8192 rows:
  // 97 / 86 / 103 us.)
  static constexpr bool kOnce = WC == 16;
  // O and the sums of the waves that share keys are joined in LDS.
  static constexpr int kPart = (4 * NF + 2) * 64;  // floats per wave
  static constexpr int kMergeB = (WK - 1) * WQ * kPart * 4;
  static constexpr int kLds = 2 * RING * kTileB > kMergeB ? 2 * RING * kTileB : kMergeB;
  // Blocks per CU: 160 KiB of LDS, and registers for 16, 8 or 4 waves.
  static constexpr int kLdsBlocks = 160 * 1024 / kLds;
  static constexpr int kWaveBlocks = (DP == 64 && !kPipe ? 16 : DP == 256 && WC == 32 ? 4 : 8) / NW;
  static constexpr int kPerCu = kLdsBlocks < kWaveBlocks ? kLdsBlocks : kWaveBlocks;
  static_assert(WC == 32 || WC == 16, "MFMA shapes");
  static_assert(BK % (KG * WK) == 0 && kIW >= 1 && kCols % 32 == 0, "tiles split evenly");
  static_assert(KG == 32 || (WC == 16 && KG == 16 && sizeof(T) == 4), "16-bit products take 32 keys");
  // The rows a wave loads lie in one 32-row group of the tile, so a page of
  // 32 rows or more is looked up once per wave and tile.
  static_assert(BK / NW <= 32 && 32 % (BK / NW) == 0, "a wave's rows share a page");
};

// Swizzles (16-byte unit u of row r is stored at u ^ swz), which spread what
// the lanes of a read take over the banks.  K: one unit each of 16 or 32
// rows.  16-bit V: transposing reads of two or four units each of 16 or 8
// rows.  Float V: 64 or 128 bytes each of rows four apart.
template <typename S>
__device__ __forceinline__ int k_swz(int r) {
  return S::kRowB >= 256 ? (r & 15) : (r & 7);
}
template <typename S>
__device__ __forceinline__ int v_swz(int r) {
  if (sizeof(typename S::T) == 4) return 4 * ((r >> 2) & 3);
  if (S::WC == 32) return S::kRowB >= 256 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
  return S::kRowB >= 256 ? (((r & 7) << 1) | ((r >> 3) & 1)) : (r & 7);
}

// One unit step of S^T: keys of `ka` against the column's `q`.
template <int WC, typename Unit, typename Acc>
__device__ __forceinline__ Acc score_step(Unit ka, Unit q, Acc s) {
  if constexpr (sizeof(ka[0]) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (WC == 32)
        s = mfma32x32x2(ka[e], q[e], s);
      else
        s = mfma16x16x4(ka[e], q[e], s);
    }
    return s;
  } else if constexpr (WC == 32) {
    return mfma32x32x16(ka, q, s);
  } else {
    return mfma16x16x32(ka, q, s);
  }
}

// Which of the 32 keys from `key0` a column sees, one bit each: mask words
// of its draft, all ones before the prefix ends, none at or past `end`.
__device__ __forceinline__ uint32_t seen_bits(const uint32_t* mask, int words, int P, int end,
                                              int key0, bool live) {
  if (!live || key0 >= end) return 0u;
  uint32_t bits = 0xffffffffu;
  const int off = key0 - P;
  if (off + 31 >= 0) {
    const int w = off >> 5;
    const uint32_t lo = w < 0 ? 0xffffffffu : (w < words ? mask[w] : 0u);
    const uint32_t hi = w + 1 < words ? mask[w + 1] : 0u;
    bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (off & 31));
  }
  const int left = end - key0;
  return left < 32 ? bits & ((1u << left) - 1u) : bits;
}

// Waits until at most N of this wave's loads are on their way.  The direct
// loads are unknown to the compiler; loads of its own among them only make
// the wait longer.
template <int N>
__device__ __forceinline__ void wait_tiles() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
#endif
}

template <typename T>
__device__ __forceinline__ bool finite(T x) {
  return fabsf(to_f32(x)) < INFINITY;
}

// Weight of a part whose reference is m in a sum whose reference is M.  A
// part that saw no row has sums of 0 (and one whose every score was a NaN
// keeps its NaN).
__device__ __forceinline__ float weight(float m, float M) {
  return m == -INFINITY ? 1.f : fast_exp2(m - M);
}

// What a gate lets through: the same form wherever a value is stored, the one
// of the prefill's.
template <typename T>
__device__ __forceinline__ float gate_weight(T g) {
  if constexpr (std::is_same<T, float>::value)
    return stable_sigmoid(g);
  else
    return fast_sigmoid(to_f32(g));
}

template <typename TO>
__device__ __forceinline__ void store4(void* out, int64_t at, const float (&r)[4], int n,
                                       bool vec) {
  TO* p = (TO*)out + at;
  if (vec && n >= 4) {
    typedef TO T4 __attribute__((ext_vector_type(4)));
    *(T4*)p = (T4){from_f32<TO>(r[0]), from_f32<TO>(r[1]), from_f32<TO>(r[2]), from_f32<TO>(r[3])};
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = from_f32<TO>(r[i]);
}

// Output channels d0 .. d0 + 3 of row `row` = (b, draft, head): the gate,
// then the one rounding.  `sees`: the draft sees a row; one that sees none
// gets zeros whatever its gate holds.
template <typename T>
__device__ __forceinline__ void write4(const TreeArgs& a, int64_t row, int d0, float (&r)[4],
                                       bool sees) {
  const int n = a.value_dim - d0;
  if (n <= 0) return;
  const int64_t at = row * a.value_dim + d0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = sees ? r[i] : 0.f;
  if (a.gate != nullptr && sees) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) r[i] *= gate_weight(((const T*)a.gate)[at + i]);
  }
  switch (a.out_dtype) {
    case ALPX_F32: store4<float>(a.out, at, r, n, a.vec_o); break;
    case ALPX_F16: store4<f16_t>(a.out, at, r, n, a.vec_o); break;
    default: store4<bf16_t>(a.out, at, r, n, a.vec_o); break;
  }
}

// The 16 bytes of a row of `width` from channel d on, zeros past its end.
template <typename T>
__device__ __forceinline__ auto row_unit(const T* row, int d, int width, bool vec) {
  constexpr int EPU = 16 / (int)sizeof(T);
  typedef T Unit __attribute__((ext_vector_type(EPU)));
  Unit x = {};
  if (vec) {
    if (d < width) x = *(const Unit*)(row + d);
  } else {
    for (int e = 0; e < EPU; ++e)
      if (d + e < width) x[e] = row[d + e];
  }
  return x;
}

// The output of columns 32 cg + 0 .. 31 and channels 32 mb + 0 .. 31 of a
// sequence whose V holds an infinity or a NaN.  The products take every row
// of a tile for every column, and 0 times either is a NaN, whether the column
// does not see the row or its weight is below the smallest number.  Here V
// enters the product with its infinities and NaN replaced by zeros, and those
// are counted apart, for each column among the rows that it sees: products of
// 0 / 1 matrices again, in the tiles that hold any.  An infinity that a column
// sees comes out as itself however small its weight (a NaN where the weight is
// exactly 0: a score of -inf).  One infinity in a prefix, one kv head of one
// sequence: 4 x 64 drafts on 32768 rows, 256 wide, 200 us -> 3.0 ms (every
// head's: 5.8), 16 x 16 on 8192, 128 wide, 97 us -> 0.55 ms; row by row, with
// one column a thread, it took 135 (494) and 18 ms.
//
// Waves 0 to 3 take 16 columns each, two of them every other 32 rows, operands
// straight from memory (few registers: the kernels that call this keep what
// their own loops need).  Every thread of the block calls it; those past 256
// only meet the barriers.  `part`: kApart floats of LDS.
constexpr int kApart = 4 * 11 * 64;
template <typename T>
__device__ __forceinline__ void set_apart(const TreeArgs& a, int b, int kvh, int cg, int mb, int P,
                                          int end, float* part) {
  constexpr int EPU = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63, cl = lane & 15, sub = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group, col = 32 * cg + 16 * (w & 1) + cl, node = col / G;
  const bool in_range = node < a.nodes, live = node < end - P;
  const int64_t row = ((int64_t)b * a.nodes + (in_range ? node : 0)) * a.q_heads + kvh * G +
                      (col - node * G);
  if (w < 4) {
    const T* q = (const T*)a.q + row * a.key_dim;
    const uint32_t* mask = a.masks + b * a.mask_b + (int64_t)(in_range ? node : 0) * a.words;
    f32x4 o[2] = {};  // channels 16 n + 4 sub + 0 .. 3 of the 32
    uint32_t found = 0;  // infinities seen: bit 4 n + i for inf, 8 + 4 n + i for -inf
    float m = -INFINITY, l = 0.f;
#pragma clang loop unroll(disable)
    for (int j0 = 32 * (w >> 1); j0 < end; j0 += 64) {
      int64_t ko = (int64_t)b * a.ks_b + j0 * a.ks_pos, vo = (int64_t)b * a.vs_b + j0 * a.vs_pos;
      if (a.pages != nullptr) {  // (a page holds whole groups of 32 rows)
        int pg = load_const(a.pages + (int64_t)b * a.max_pages + (j0 >> a.page_shift));
        pg = min(max(pg, 0), a.num_pages - 1);
        const int64_t in = j0 & ((1 << a.page_shift) - 1);
        ko = pg * a.ks_b + in * a.ks_pos;
        vo = pg * a.vs_b + in * a.vs_pos;
      }
      const int rows = end - j0;
      const T* k = (const T*)a.k + ko + (int64_t)kvh * a.ks_h;
      const T* v = (const T*)a.v + vo + (int64_t)kvh * a.vs_h;
      // (32 rows lie within 2^31 bytes)
      const T* k0 = k + min(cl, rows - 1) * (uint32_t)a.ks_pos;
      const T* k1 = k + min(16 + cl, rows - 1) * (uint32_t)a.ks_pos;
      f32x4 sc[2] = {};
      for (int d0 = 0; d0 < a.key_dim; d0 += 4 * EPU) {
        const int d = d0 + EPU * sub;
        const auto qd = row_unit(q, d, a.key_dim, a.vec_q);
        sc[0] = score_step<16>(row_unit(k0, d, a.key_dim, a.vec_k), qd, sc[0]);
        sc[1] = score_step<16>(row_unit(k1, d, a.key_dim, a.vec_k), qd, sc[1]);
      }
      // score r is of key 16 (r / 4) + 4 sub + r % 4
      const uint32_t seen = seen_bits(mask, a.words, P, end, j0, live) >> (4 * sub);
      float s[8], mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const bool keep = seen >> (16 * (r >> 2) + (r & 3)) & 1;
        s[r] = keep ? sc[r >> 2][r & 3] * a.scale_log2 : -INFINITY;
        // (the reference is finite from the first row that is seen)
        if (keep) mx = fmaxf(mx, fmaxf(s[r], -__FLT_MAX__));
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
      const float c = weight(m, mx), off = mx == -INFINITY ? 0.f : mx - kLift<T>;
      m = mx;
      l *= c;
      uint32_t none = 0;  // rows that are seen without weight
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (s[r] == -INFINITY) none |= seen & 1u << (16 * (r >> 2) + (r & 3));
        s[r] = fast_exp2(s[r] - off);
        l += s[r];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        // x[r]: this lane's channel 16 n + cl of the key of score r
        const int channel = 32 * mb + 16 * n + cl;
        float x[8];
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int key = 16 * (r >> 2) + 4 * sub + (r & 3);
          x[r] = to_f32(v[min(key, rows - 1) * (uint32_t)a.vs_pos + min(channel, a.value_dim - 1)]);
          if (key >= rows) x[r] = 0.f;
          odd |= !finite(x[r]);
        }
        // the product of f(r).first at key and channel, f(r).second at key and column
        typedef std::pair<float, float> Two;
        auto product = [&](auto f, f32x4 acc) __attribute__((always_inline)) {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int r = 0; r < 8; ++r) acc = mfma16x16x4(f(r).first, f(r).second, acc);
          } else {
            typename Vec8<T>::type xs, ps;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              xs[r] = from_f32<T>(f(r).first);
              ps[r] = from_f32<T>(f(r).second);
            }
            acc = mfma16x16x32(xs, ps, acc);
          }
          return acc;
        };
        o[n] = product([&](int r) { return Two(finite(x[r]) ? x[r] : 0.f, s[r]); }, o[n] * c);
        if constexpr (sizeof(T) == 2)  // P in two parts, as in the narrow kernels
          o[n] = product([&](int r) {
            return Two(finite(x[r]) ? x[r] : 0.f, s[r] - to_f32(from_f32<T>(s[r])));
          }, o[n]);
        if (__ballot(odd) == 0) continue;
        // a row that is seen counts an infinity of its sign, and a NaN as
        // both; one without weight counts either as both
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {
          const float other = sign == 0 ? -INFINITY : INFINITY;
          f32x4 count = product([&](int r) {
            return Two(finite(x[r]) || x[r] == other ? 0.f : 1.f,
                       (float)(seen >> (16 * (r >> 2) + (r & 3)) & 1));
          }, (f32x4)(0.f));
          count = product([&](int r) {
            return Two(x[r] == other ? 1.f : 0.f, (float)(none >> (16 * (r >> 2) + (r & 3)) & 1));
          }, count);
#pragma unroll
          for (int i = 0; i < 4; ++i) found |= (uint32_t)(count[i] > 0.f) << (8 * sign + 4 * n + i);
        }
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float* to = part + w * 11 * 64 + lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i * 64] = o[i >> 2][i & 3];
    to[8 * 64] = m;
    to[9 * 64] = l;
    to[10 * 64] = __uint_as_float(found);
  }
  __syncthreads();
  if (w < 4 && in_range) {  // wave w writes channels 16 n + 4 sub + 0 .. 3 of its columns
    const int n = w >> 1;
    const float* p0 = part + (w & 1) * 11 * 64 + lane;
    const float* p1 = p0 + 2 * 11 * 64;
    const float m0 = p0[8 * 64], m1 = p1[8 * 64], M = fmaxf(m0, m1);
    const float c0 = weight(m0, M), c1 = weight(m1, M);
    const float l = p0[9 * 64] * c0 + p1[9 * 64] * c1;
    const uint32_t found = __float_as_uint(p0[10 * 64]) | __float_as_uint(p1[10 * 64]);
    const float inv = l == 0.f ? NAN : 1.f / l;  // (rows that all score -inf: 0 / 0)
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * n + i;
      r[i] = (p0[at * 64] * c0 + p1[at * 64] * c1) * inv;
      if (found >> at & 1) r[i] += INFINITY;
      if (found >> (8 + at) & 1) r[i] -= INFINITY;
    }
    write4<T>(a, row, 32 * mb + 16 * n + 4 * sub, r, M != -INFINITY);
  }
  __syncthreads();  // `part` is read
}

// One block: slot `s`, kv head and column tile; it walks its run of tiles,
// sequence by sequence.  ALONE: slot `s` is sequence `s`.
//
// Lane (cl, sub) of a wave owns column cl and, of every 4 LPC keys or
// channels, the four from 4 sub on: the order in which an MFMA leaves its
// result.  Both products take their inner index in that order too, so the
// probabilities are an operand where they lie.
template <typename S, bool DMA, bool ALONE>
__global__ void __launch_bounds__(64 * S::NW, S::kPerCu* S::NW / 4) tree_kernel(TreeArgs a) {
  static_assert(!ALONE || (S::kLds >= kApart * 4 && S::NW >= 4), "set_apart's space and threads");
  typedef typename S::T T;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int BK = S::BK, WC = S::WC, LPC = S::LPC, KG = S::KG, EPU = S::EPU, U = S::U;
  constexpr int NF = S::NF, NS = S::NS, NQ = S::NQ, kRowB = S::kRowB, kTileB = S::kTileB;
  constexpr int DB = WC;             // channels of one MFMA of O^T
  constexpr int NB = S::DP / DB;     // such blocks
  constexpr int KB = WC == 32 ? 1 : KG / 16;  // MFMA blocks of a key group
  typedef T Unit __attribute__((ext_vector_type(EPU)));
  typedef typename std::conditional<WC == 32, f32x16, f32x4>::type Acc;
  constexpr int NA = WC == 32 ? 16 : 4;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLds];  // K 0, V 0, K 1, V 1, ..

  const int tid = threadIdx.x, thread_lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave % S::WK, wq = wave / S::WK;  // a column's waves on different SIMDs
  const int G = a.group;

  // The column tiles of one (slot, kv head) run next to each other on one
  // XCD, whose L2 then holds the tiles that they all read.
  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds;
  const int ct = at % a.col_tiles;
  const int unit = (at / a.col_tiles) * kXcds + xcd;
  const int slot = unit / a.kv_heads, kvh = unit % a.kv_heads;
  if (slot >= a.slots) return;
  Share sh;
  if constexpr (ALONE) {  // a slot per sequence
    sh = {};
    sh.b = slot;
    uniform_rows(a, slot, sh.P, sh.end);
    sh.tiles = sh.nt = (sh.end + BK - 1) / BK;
  } else {
    sh = find_share<BK>(a, slot, unit == 0 && ct == 0 && wave == 0);
    if (sh.b < 0) return;  // fewer tiles than slots
  }

  // Tile loads: wave w fills rows [w BK / NW, (w + 1) BK / NW) of a tile, all
  // in its 32-row group `grp`.
  constexpr int kRows = BK / S::NW;
  const int grp = wave * kRows / 32 * 32;
  uint32_t kofs[S::kIW], vofs[S::kIW];
#pragma unroll
  for (int i = 0; i < S::kIW; ++i) {
    const int sl = (wave * S::kIW + i) * 64 + thread_lane;
    const int r = sl / U;
    const int uk = (sl % U) ^ k_swz<S>(r), uv = (sl % U) ^ v_swz<S>(r);
    // units past the head width: an offset past every row, which reads zero
    kofs[i] = uk * EPU < a.key_dim
                  ? (uint32_t)(((int64_t)(r - grp) * a.ks_pos + EPU * uk) * (int64_t)sizeof(T))
                  : 0x80000000u;
    vofs[i] = uv * EPU < a.value_dim
                  ? (uint32_t)(((int64_t)(r - grp) * a.vs_pos + EPU * uv) * (int64_t)sizeof(T))
                  : 0x80000000u;
  }
  const uint32_t lbase = (uint32_t)(uintptr_t)(lds_void_t*)smem;

  for (;;) {
    // opaque, so that nothing formed from it is kept over the tile loop for
    // the next sequence (those values took the registers of the loop)
    int lane = thread_lane;
    pin(lane);
    const int cl = lane % WC, sub = lane / WC;
    const int col = ct * S::kCols + WC * wq + cl;
    const int node = col / G;
    const bool in_range = node < a.nodes;
    const int b = sh.b, P = sh.P;
    const int t0 = sh.t0, nt = sh.nt;
    if (!ALONE && t0 == 0 && kvh == 0 && ct == 0 && tid == 0)
      a.found[b] = make_int4(slot, sh.s1, P, sh.end);
    bool again = false;  // alone: some of the output is not finite
    auto segment = [&]() __attribute__((always_inline)) {
      // rows [start, stop) of sequence b, in tiles of BK: none where no column
      // of the block has a draft
      const int count = sh.end - P;
      const bool none = ct * S::kCols >= count * G;
      if (none && (nt < sh.tiles || !a.direct)) return;
      const int turns = none ? 0 : nt;
      const int start = t0 * BK, stop = none ? start : min(sh.end, start + nt * BK);
      const bool live = node < count;
      // a wave without a live column only loads and meets the barriers
      const bool idle = ct * S::kCols + WC * wq >= count * G;
      const int64_t qrow = ((int64_t)b * a.nodes + (in_range ? node : 0)) * a.q_heads + kvh * G +
                           (col - node * G);
      const uint32_t* mask = a.masks + b * a.mask_b + (int64_t)(in_range ? node : 0) * a.words;

      auto group_base = [&](int row, const T*& kb, const T*& vb) __attribute__((always_inline)) {
        if (a.pages != nullptr) {
          int pg = load_const(a.pages + (int64_t)b * a.max_pages + (row >> a.page_shift));
          pg = min(max(pg, 0), a.num_pages - 1);
          const int64_t in = row & ((1 << a.page_shift) - 1);
          kb = (const T*)a.k + pg * a.ks_b + in * a.ks_pos + (int64_t)kvh * a.ks_h;
          vb = (const T*)a.v + pg * a.vs_b + in * a.vs_pos + (int64_t)kvh * a.vs_h;
        } else {
          kb = (const T*)a.k + (int64_t)b * a.ks_b + (int64_t)row * a.ks_pos + (int64_t)kvh * a.ks_h;
          vb = (const T*)a.v + (int64_t)b * a.vs_b + (int64_t)row * a.vs_pos + (int64_t)kvh * a.vs_h;
        }
      };
      // Where tile t's K and V lie; rows past the end (all of them past the
      // last tile) read as zeros, or, where rows lie over each other, as what
      // the rows before hold there (no column sees them).
      struct Source {
        const T *k, *v;
        int rows;
        i32x4 rk, rv;
      };
      auto source = [&](int t) __attribute__((always_inline)) {
        Source s;
        const int row0 = start + t * BK + grp;
        s.rows = __builtin_amdgcn_readfirstlane(min(max(stop - row0, 0), 32));
        s.k = (const T*)a.k;
        s.v = (const T*)a.v;
        if (s.rows > 0) group_base(row0, s.k, s.v);
        // to the last row's last value, since rows may lie over each other
        // (32 rows lie within 2^31 bytes)
        auto bytes = [&](int64_t pitch, int width) __attribute__((always_inline)) {
          return s.rows > 0 ? ((s.rows - 1) * (uint32_t)pitch + width) * (uint32_t)sizeof(T) : 0u;
        };
        s.rk = rsrc_words((uint64_t)(uintptr_t)s.k, bytes(a.ks_pos, a.key_dim));
        s.rv = rsrc_words((uint64_t)(uintptr_t)s.v, bytes(a.vs_pos, a.value_dim));
        return s;
      };
      // load i of this wave's share of a K (V) tile, to LDS byte dst
      auto load_k = [&](const Source& s, int i, uint32_t dst) __attribute__((always_inline)) {
        lds_dma16(s.rk, lbase + dst + (wave * S::kIW + i) * 1024, kofs[i]);
      };
      auto load_v = [&](const Source& s, int i, uint32_t dst) __attribute__((always_inline)) {
        if (S::kOnce)
          lds_dma16_once(s.rv, lbase + dst + (wave * S::kIW + i) * 1024, vofs[i]);
        else
          lds_dma16(s.rv, lbase + dst + (wave * S::kIW + i) * 1024, vofs[i]);
      };
      auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
        const Source s = source(t);
        const uint32_t dst = buf * 2 * kTileB;
        if constexpr (DMA) {
#pragma unroll
          for (int i = 0; i < S::kIW; ++i) load_k(s, i, dst);
#pragma unroll
          for (int i = 0; i < S::kIW; ++i) load_v(s, i, dst + kTileB);
        } else {
          // any head width, stride or alignment: element by element, through
          // registers (4 x 8 drafts on 4096 rows: 33 wide bf16 43.6 us,
          // float32 60.2, against 18.5 and 27.4 for rows of 40 and 36 by
          // direct loads; 100 wide bf16 76, 104 wide 25; 250 wide 52, 248 26)
          for (int i = lane; i < kRows * S::DP; i += 64) {
            const int r = wave * kRows + i / S::DP, d = i % S::DP;
            const int64_t row = r - grp;
            const bool in = row < s.rows;
            const T kx = in && d < a.key_dim ? s.k[row * a.ks_pos + d] : from_f32<T>(0.f);
            const T vx = in && d < a.value_dim ? s.v[row * a.vs_pos + d] : from_f32<T>(0.f);
            const int u = d / EPU, e = d % EPU;
            T* k = (T*)(smem + dst);
            k[r * S::DP + (u ^ k_swz<S>(r)) * EPU + e] = kx;
            k[kTileB / (int)sizeof(T) + r * S::DP + (u ^ v_swz<S>(r)) * EPU + e] = vx;
          }
        }
      };

      // the ring's first tiles, the queries while they are on their way
      if constexpr (S::kPipe) {
        const Source s0 = source(0), s1 = source(1);
#pragma unroll
        for (int i = 0; i < S::kIW; ++i) load_k(s0, i, 0);
#pragma unroll
        for (int i = 0; i < S::kIW; ++i) load_k(s1, i, kTileB);
      } else {
#pragma unroll
        for (int i = 0; i < S::RING - 1; ++i) load_tile(i, i);
      }
      // B operand of S^T: this lane's units of its column's query row (unit
      // LPC j + sub), zero past the head width.
      Unit qv[NQ];
      {
        const T* qp = (const T*)a.q + qrow * a.key_dim;
        // channels past the width: the last ones again, their bits cleared
        const int on = live ? -1 : 0;
        if (a.vec_q) {
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            const int d = EPU * (LPC * j + sub);
            const u32x4 x = *(const u32x4*)(qp + min(d, a.key_dim - EPU));
            qv[j] = __builtin_bit_cast(Unit, x & (uint32_t)(on & ((d - a.key_dim) >> 31)));
          }
        } else {
          typedef typename std::conditional<F32, int32_t, int16_t>::type Bits;
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
#pragma unroll
            for (int e = 0; e < EPU; ++e) {
              const int d = EPU * (LPC * j + sub) + e;
              const Bits x = __builtin_bit_cast(Bits, qp[min(d, a.key_dim - 1)]);
              qv[j][e] = __builtin_bit_cast(T, (Bits)(x & on & ((d - a.key_dim) >> 31)));
            }
          }
        }
      }

      Acc o[NB];              // O^T[channel DB n + 4 LPC (r / 4) + 4 sub + r % 4][column]
      float m = -INFINITY;    // the column's reference score
      float l = 0.f;          // this lane's share of the sum of P
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n] = (Acc)(0.f);
      if constexpr (S::kPipe) {
        // Turn t: PV of tile t - 1, the softmax of tile t and QK of tile
        // t + 1, so that the products run beside the exponentials of the same
        // wave, while K of tile t + 2 and V of tile t are on their way.  The
        // first turn has no PV, the last one (turn `turns`) nothing else.  K tiles
        // at 0 and kTileB, V tiles at 2 and 3 kTileB.
        typedef typename Vec8<T>::type V8;
        typedef typename Vec4<T>::type V4;
        constexpr int KR = S::KR, NV = 2 * KR * NB, NK = KR * NQ, NE = 16 * KR;
        Acc sc[KR];
        V8 pv[2 * KR];
        float pend = 1.f;  // what O still has to be multiplied by
        bool pend_any = false;
        // byte offsets of this lane's operands: K row cl of a group, unit
        // 2 j + sub (16 units on: 256 bytes); V row 4 sub + (lane % 16) / 4
        // of 8, channels 32 n + 16 ((lane / 16) % 2) + 4 (lane % 4)
        constexpr int KA = NQ < 8 ? NQ : 8, VA = NB < 4 ? NB : 4;
        int kadr[KA], vadr[VA];
        const int vrow = 4 * sub + ((lane & 15) >> 2);
#pragma unroll
        for (int j = 0; j < KA; ++j) kadr[j] = cl * kRowB + ((2 * j + sub) ^ k_swz<S>(cl)) * 16;
#pragma unroll
        for (int n = 0; n < VA; ++n)
          vadr[n] = 2 * kTileB + vrow * kRowB +
                    ((4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swz<S>(vrow)) * 16 +
                    8 * (lane & 1);
        auto k_operand = [&](int buf, int kr, int j) __attribute__((always_inline)) {
          return *(const Unit*)(smem + kadr[j % KA] + buf + 32 * kr * kRowB + j / KA * 256);
        };
        auto v_operand = [&](int buf, int ks, int n) __attribute__((always_inline)) {
          const char* p = smem + vadr[n % VA] + buf + 16 * ks * kRowB + n / VA * 256;
          const V4 x0 = lds_read_tr4((const T*)p), x1 = lds_read_tr4((const T*)(p + 8 * kRowB));
          return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
#pragma unroll
        for (int kr = 0; kr < KR; ++kr) {
          sc[kr] = (Acc)(0.f);
#pragma unroll
          for (int j = 0; j < NQ; ++j) sc[kr] = mfma32x32x16(k_operand(0, kr, j), qv[j], sc[kr]);
        }
        __syncthreads();  // K 0 is read before turn 0 refills it
        auto turn = [&](auto parity, auto place, int t) __attribute__((always_inline)) {
          constexpr int Q = decltype(parity)::value;  // t & 1, but for the last
          constexpr bool FIRST = decltype(place)::value == 0, LAST = decltype(place)::value == 2;
          // the other place of each pair: tile t - 1 of V, tile t + 1 of K
          const int behind = LAST ? ((turns & 1) ^ 1) * kTileB : (Q ^ 1) * kTileB;
          // the turn's loads (past the last tile they fetch nothing and write
          // zeros where nothing is read): spread over the steps, since a wave
          // that issues them in one go waits for the address unit meanwhile
          constexpr int NL = LAST ? 0 : S::kTileLoads;
          Source sk, sv;
          if constexpr (!LAST) {
            sk = source(t + 2);
            sv = source(t);
          }
          auto load = [&](int i) __attribute__((always_inline)) {
            if (i < S::kIW)
              load_v(sv, i, (2 + Q) * kTileB);
            else
              load_k(sk, i - S::kIW, Q * kTileB);
          };
          if (idle) {
#pragma unroll
            for (int i = 0; i < NL; ++i) load(i);
          } else {
            // O holds tiles up to t - 2 and is about to take P of tile t - 1,
            // formed against the reference that moved there
            if (__builtin_expect(pend_any, 0)) {
#pragma unroll
              for (int n = 0; n < NB; ++n) o[n] *= pend;
              pend = 1.f;
              pend_any = false;
            }
            const int key0 = start + t * BK;
            if (!LAST && key0 + BK > P) {  // not all of these keys are prefix rows
#pragma unroll
              for (int kr = 0; kr < KR; ++kr) {
                const uint32_t mine =
                    seen_bits(mask, a.words, P, stop, key0 + 32 * kr, live) >> (4 * sub);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const int keep = (int)(mine << (31 - (8 * (r >> 2) + (r & 3)))) >> 31;
                  sc[kr][r] = __int_as_float((__float_as_int(sc[kr][r]) & keep) |
                                             (0xff800000 & ~keep));
                }
              }
            }
            if constexpr (!LAST) {
              float mx = sc[0][0];
#pragma unroll
              for (int r = 1; r < NE; ++r) mx = fmaxf(mx, sc[r / 16][r % 16]);
              mx *= a.scale_log2;
              if (__builtin_expect(__ballot(mx > m + kRescale) != 0, 0)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                if (mx > m + kRescale) {
                  pend = fast_exp2(m - mx);
                  l *= pend;
                  m = mx;
                }
                pend_any = true;
              }
            }
            const float off = m == -INFINITY ? 0.f : m - kLift<T>;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            float ps = 0.f;
            V8 pn[2 * KR];
            auto probability = [&](auto e_) __attribute__((always_inline)) {
              constexpr int e = decltype(e_)::value;
              const float p = fast_exp2(fmaf(sc[e / 16][e % 16], a.scale_log2, -off));
              ps += p;
              pn[e / 8][e % 8] = from_f32<T>(p);
            };
            if constexpr (FIRST) static_for<0, NE>(probability);
            // P is rounded to the cache's type for its product, as the
            // prefill's: these kernels are bound by the products (the rest of
            // P as a second one: 4 x 63 on 4133 rows, 128 wide, 28.9 -> 32.0
            // us, 4 x 64 on 32768, 256 wide, 152 -> 185).
            // Step i: product i of NP + NS and its share of the exponentials,
            // all of them before their registers take tile t + 1's scores.
            // Operands are read AHEAD steps before their product; the order
            // is kept as written (left to itself the scheduler reads each
            // operand right before its product and waits for it).
            constexpr int NP = FIRST ? 0 : NV, N = NP + (LAST ? 0 : NK), AHEAD = 4;
            constexpr int BY = NP + (KR - 1) * NQ;  // the exponentials' last step
            u32x4 opd[N];
            auto read = [&](auto i_) __attribute__((always_inline)) {
              constexpr int i = decltype(i_)::value;
              if constexpr (i < NP)
                opd[i] = __builtin_bit_cast(u32x4, v_operand(behind, i / NB, i % NB));
              else
                opd[i] = __builtin_bit_cast(
                    u32x4, k_operand(behind, (i - NP) / NQ, (i - NP) % NQ));
            };
            static_for<0, AHEAD>(read);
            static_for<0, N>([&](auto i_) __attribute__((always_inline)) {
              constexpr int i = decltype(i_)::value;
              if constexpr (i + AHEAD < N) read(Par<i + AHEAD>());
              const V8 x = __builtin_bit_cast(V8, opd[i]);
              if constexpr (i < NP) {
                o[i % NB] = mfma32x32x16(x, pv[i / NB], o[i % NB]);
              } else {
                constexpr int kr = (i - NP) / NQ, j = (i - NP) % NQ;
                if constexpr (j == 0)
                  sc[kr] = mfma32x32x16(x, qv[j], (Acc)(0.f));
                else
                  sc[kr] = mfma32x32x16(x, qv[j], sc[kr]);
              }
              // loads first, in the steps' first three quarters
              constexpr int d0 = i * NL * 4 / (3 * N), d1 = (i + 1) * NL * 4 / (3 * N);
              static_for<(d0 < NL ? d0 : NL), (d1 < NL ? d1 : NL)>(
                  [&](auto d_) __attribute__((always_inline)) { load(decltype(d_)::value); });
              if constexpr (!FIRST && !LAST)
                static_for<(i < BY ? i * NE / BY : NE), (i + 1 < BY ? (i + 1) * NE / BY : NE)>(
                    probability);
              __builtin_amdgcn_sched_barrier(0);
            });
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!LAST) {
              l += ps;
#pragma unroll
              for (int i = 0; i < 2 * KR; ++i) {
                pv[i] = pn[i];
                pin(pv[i]);
              }
            }
          }
          if constexpr (!LAST) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
          }
        };
        turn(Par<0>(), Par<0>(), 0);
#pragma clang loop unroll(disable)
        for (int t = 1; t < turns; t += 2) {
          turn(Par<1>(), Par<1>(), t);
          if (t + 1 < turns) turn(Par<0>(), Par<1>(), t + 1);
        }
        turn(Par<0>(), Par<2>(), turns);
      } else {
        wait_tiles<(S::RING - 2) * S::kTileLoads * DMA>();  // the first tile is in LDS
        __syncthreads();
        int buf = 0;
#pragma clang loop unroll(disable)
        for (int t = 0; t < turns; ++t) {
          // into the place of the tile before this one; past the last tile the
          // loads fetch nothing and write zeros, so that every turn waits for
          // the same number
          load_tile(t + S::RING - 1, buf == 0 ? S::RING - 1 : buf - 1);
          const char* kt = smem + buf * 2 * kTileB;
          const char* vt = kt + kTileB;
          if (!idle) {
            const int g0 = KG * S::KR * wk;  // this wave's keys of the tile
            const int key0 = start + t * BK + g0;
            // All of them through each step together, so that one group's
            // products run beside the other's softmax.
            Acc sa[S::KR * KB];
#pragma unroll
            for (int kb = 0; kb < S::KR * KB; ++kb) sa[kb] = (Acc)(0.f);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
              for (int kb = 0; kb < S::KR * KB; ++kb) {
                const int row = g0 + WC * kb + cl;
                const Unit ka =
                    *(const Unit*)(kt + row * kRowB + ((LPC * j + sub) ^ k_swz<S>(row)) * 16);
                sa[kb] = score_step<WC>(ka, qv[j], sa[kb]);
              }
            constexpr int NT = S::KR * NS;
            float s[NT];  // score r is of key g0 + 4 LPC (r / 4) + 4 sub + r % 4
#pragma unroll
            for (int r = 0; r < NT; ++r) s[r] = sa[r / NA][r % NA];
            if (key0 + KG * S::KR > P) {  // not all of these keys are prefix rows
#pragma unroll
              for (int kr = 0; kr < S::KR; ++kr) {
                const uint32_t mine =
                    seen_bits(mask, a.words, P, stop, key0 + KG * kr, live) >> (4 * sub);
#pragma unroll
                for (int r = 0; r < NS; ++r) {
                  // all bits or none
                  const int keep = (int)(mine << (31 - (4 * LPC * (r >> 2) + (r & 3)))) >> 31;
                  float& x = s[kr * NS + r];
                  x = __int_as_float((__float_as_int(x) & keep) | (0xff800000 & ~keep));
                }
              }
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < NT; ++r) mx = fmaxf(mx, s[r]);
            mx *= a.scale_log2;
            // the reference moves only when a score exceeds it by more than
            // kRescale, so P <= 2^kRescale and the sums keep their range
            if (__ballot(mx > m + kRescale) != 0) {
              if constexpr (LPC == 4) mx = fmaxf(mx, __shfl_xor(mx, 16));
              mx = fmaxf(mx, __shfl_xor(mx, 32));
              if (mx > m + kRescale) {
                const float c = fast_exp2(m - mx);  // 0 while m is -inf
                l *= c;
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] *= c;
                m = mx;
              }
            }
            const float off = m == -INFINITY ? 0.f : m - kLift<T>;
            float ps = 0.f;
#pragma unroll
            for (int kr = 0; kr < S::KR; ++kr) {
              float* p_ = s + kr * NS;
#pragma unroll
              for (int r = 0; r < NS; ++r) {
                p_[r] = fast_exp2(fmaf(p_[r], a.scale_log2, -off));
                ps += p_[r];
              }
              if constexpr (F32) {
#pragma unroll
                for (int r = 0; r < NS; ++r) {
                  const int vr = g0 + KG * kr + 4 * LPC * (r >> 2) + 4 * sub + (r & 3);
#pragma unroll
                  for (int n = 0; n < NB; ++n) {
                    const int u = (DB * n + cl) / 4;
                    const float x =
                        *(const float*)(vt + vr * kRowB + (u ^ v_swz<S>(vr)) * 16 + 4 * (cl & 3));
                    if constexpr (WC == 32)
                      o[n] = mfma32x32x2(x, p_[r], o[n]);
                    else
                      o[n] = mfma16x16x4(x, p_[r], o[n]);
                  }
                }
              } else {
                static_assert(WC == 16, "32 columns of 16 bits run the turns above");
                typedef typename Vec8<T>::type V8;
                typedef typename Vec4<T>::type V4;
#pragma unroll
                for (int ks = 0; ks < NS / 8; ++ks) {
                  // P enters its product in two parts, rounded and the rest:
                  // rounded alone it was as far off as the output's rounding
                  // (bf16, rms of the result 2.3e-3, in two parts 1.67e-3, the
                  // output's share).  A product behind the other, 16 x 16
                  // drafts on 8192 rows, 128 wide: 65.2 -> 65.6 us (69 with
                  // both to an accumulator back to back); 8 x 16 on 65536, 64
                  // wide: 197 -> 198 (192 -> 200 on another card)
                  V8 p, rest;
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    p[e] = from_f32<T>(p_[8 * ks + e]);
                    rest[e] = from_f32<T>(fmaf(to_f32(p[e]), -1.f, p_[8 * ks + e]));
                  }
                  // transposing reads: lane 4 k + q of 16 supplies row k, channels
                  // 4 q .. 4 q + 3, and receives channel lane % 16 of the four rows
                  const int vr = g0 + KG * kr + 8 * LPC * ks + 4 * sub + ((lane & 15) >> 2);
                  V8 x[NB];
#pragma unroll
                  for (int n = 0; n < NB; ++n) {
                    const int u = DB / 8 * n + ((lane & 3) >> 1);
                    const T* p0 =
                        (const T*)(vt + vr * kRowB + (u ^ v_swz<S>(vr)) * 16 + 8 * (lane & 1));
                    const int vr1 = vr + 4 * LPC;
                    const T* p1 =
                        (const T*)(vt + vr1 * kRowB + (u ^ v_swz<S>(vr1)) * 16 + 8 * (lane & 1));
                    const V4 x0 = lds_read_tr4(p0), x1 = lds_read_tr4(p1);
                    x[n] = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[n] = mfma16x16x32(x[n], p, o[n]);
                  }
#pragma unroll
                  for (int n = 0; n < NB; ++n) o[n] = mfma16x16x32(x[n], rest, o[n]);
                }
              }
            }
            l += ps;
          }
          wait_tiles<(S::RING - 2) * S::kTileLoads * DMA>();  // the next tile is in LDS
          __syncthreads();
          buf = buf + 1 == S::RING ? 0 : buf + 1;
        }
      }
      __builtin_amdgcn_s_waitcnt(0);  // no load may land behind the loop
      if constexpr (S::WK > 1) __syncthreads();  // nor any other wave's

      if constexpr (LPC == 4) l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if constexpr (S::WK > 1) {
        // the waves of a column tile's keys, joined in LDS by the first of them
        float* part = (float*)smem;
        if (wk > 0) {
          float* p = part + ((wk - 1) * S::WQ + wq) * S::kPart + lane;
#pragma unroll
          for (int i = 0; i < 4 * NF; ++i) p[i * 64] = o[i / NA][i % NA];
          p[4 * NF * 64] = m;
          p[(4 * NF + 1) * 64] = l;
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int w = 0; w < S::WK - 1; ++w) {
          const float* p = part + (w * S::WQ + wq) * S::kPart + lane;
          const float m1 = p[4 * NF * 64], l1 = p[(4 * NF + 1) * 64];
          const float M = fmaxf(m, m1);
          const float c0 = weight(m, M), c1 = weight(m1, M);
          l = l * c0 + l1 * c1;
#pragma unroll
          for (int i = 0; i < 4 * NF; ++i)
            o[i / NA][i % NA] = o[i / NA][i % NA] * c0 + p[i * 64] * c1;
          m = M;
        }
      }
      // piece f of this lane: channels 4 LPC f + 4 sub + 0 .. 3
      auto piece = [&](int f) __attribute__((always_inline)) {
        const int i = 4 * f;
        return (f32x4){o[i / NA][i % NA], o[i / NA][i % NA + 1], o[i / NA][i % NA + 2],
                       o[i / NA][i % NA + 3]};
      };
      const int64_t seg = (((int64_t)(slot + b) * a.kv_heads + kvh) * a.col_tiles + ct) *
                              (S::kCols / 32) + WC * wq / 32;
      const int c32 = (WC * wq) % 32 + cl;  // column in its group of 32
      if (nt < sh.tiles || !a.direct) {
        if (idle) return;
        // [piece of 8 channels][4 of them][column]
        f32x4* po = (f32x4*)a.part_o + seg * (S::DP * 8) + c32;
#pragma unroll
        for (int f = 0; f < NF; ++f) po[(LPC * f + sub) * 32] = piece(f);
        if (sub == 0) a.part_st[seg * 32 + c32] = make_float2(m, l);
        return;
      }
      // a whole sequence: the output, and whether some of it is not finite
      float zero = 0.f;  // 0 times anything else is a NaN
#pragma unroll
      for (int i = 0; i < 4 * NF; ++i) zero = fmaf(o[i / NA][i % NA], 0.f, zero);
      // (a sum of 0: no row seen, or all of them at -inf; a sum that is a NaN
      // makes one of every channel, as it should)
      const bool bad = __ballot(live && l == l && (zero != 0.f || l == 0.f)) != 0;
      if (!ALONE && sub == 0) a.part_st[seg * 32 + c32] = make_float2(bad ? 1.f : 0.f, 0.f);
      again |= bad;
      if (!in_range) return;
      const float inv = live && l != 0.f ? 1.f / l : 0.f;
      const int64_t out0 = qrow * S::DP + 4 * sub;
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n] = live ? o[n] * inv : (Acc)(0.f);
      if (a.gate != nullptr && live) {  // the others are zeros whatever their gate holds
        typedef typename Vec4<T>::type V4;
        const T* gp = (const T*)a.gate + out0;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const V4 g = *(const V4*)(gp + 4 * LPC * f);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[4 * f / NA][4 * f % NA + i] *= gate_weight((T)g[i]);
        }
      }
      auto store = [&](auto zero_of_type) __attribute__((always_inline)) {
        typedef decltype(zero_of_type) TO;
        typedef TO TO4 __attribute__((ext_vector_type(4)));
        TO* op = (TO*)a.out + out0;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const f32x4 x = piece(f);
          *(TO4*)(op + 4 * LPC * f) = (TO4){from_f32<TO>(x[0]), from_f32<TO>(x[1]),
                                            from_f32<TO>(x[2]), from_f32<TO>(x[3])};
        }
      };
      switch (a.out_dtype) {
        case ALPX_F32: store(0.f); break;
        case ALPX_F16: store((f16_t)0.f); break;
        default: store((bf16_t)0.f); break;
      }
    };
    segment();
    if constexpr (ALONE) {
      if (__syncthreads_or(again)) {
        for (int i = 0; i < S::kCols / 32 * (S::DP / 32); ++i)
          set_apart<T>(a, b, kvh, ct * (S::kCols / 32) + i / (S::DP / 32), i % (S::DP / 32), P,
                      sh.end, (float*)smem);
      }
      return;
    }
    if (sh.left == 0) return;
    // the next sequence that has rows
    do {
      ++sh.b;
      uniform_rows(a, sh.b, sh.P, sh.end);
      sh.tiles = (sh.end + BK - 1) / BK;
    } while (sh.tiles == 0);
    sh.t0 = 0;
    sh.nt = min(sh.left, sh.tiles);
    sh.left -= sh.nt;
    sh.s1 = slot + (sh.tiles - sh.nt + sh.per - 1) / sh.per;
    __syncthreads();  // every wave is done with the tiles in LDS
  }
}

// Joins the segments of the sequences that more than one slot has tiles of,
// and writes zeros for those without a row.  One block per (sequence, kv
// head, 32 columns, 32 channels); its four waves take the segments in turn
// and meet in LDS.  A block whose result is not finite forms it again
// (set_apart).
template <typename T, int DP>
__global__ void __launch_bounds__(256) tree_join(TreeArgs a) {
  constexpr int MB = DP / 32, kFlight = 4;
  __shared__ float part[4 * 18 * 64];  // of the segments, or set_apart's
  static_assert(kApart <= 4 * 18 * 64, "set_apart's space");
  const int lane = threadIdx.x & 63, hl = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int mb = blockIdx.x % MB;
  const int groups = a.col_tiles;  // of 32 columns
  const int cg = blockIdx.x / MB % groups;
  const int kvh = blockIdx.x / MB / groups % a.kv_heads;
  const int b = blockIdx.x / MB / groups / a.kv_heads;
  const int32_t* found = (const int32_t*)(a.found + b);
  const int s0 = load_const(found), s1 = load_const(found + 1);
  const int P = load_const(found + 2), end = load_const(found + 3);
  const bool whole = a.direct && s0 == s1;  // written by its slot
  if (whole) {  // the two waves of 16 columns have a mark each
    const float2* mark = a.part_st + (((int64_t)(s0 + b) * a.kv_heads + kvh) * groups + cg) * 32;
    if (mark[0].x == 0.f && mark[16].x == 0.f) return;
  }
  const int G = a.group, col = 32 * cg + hl, node = col / G;
  const int count = end - P;
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
  if (!whole && 32 * cg < count * G) {
    for (int s = s0 + w; s <= s1; s += 4 * kFlight) {
      float2 st[kFlight];
      f32x4 x[kFlight][4];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int su = min(s + 4 * u, s1);  // past the last: its loads again, unused
        const int64_t seg = ((int64_t)(su + b) * a.kv_heads + kvh) * groups + cg;
        st[u] = a.part_st[seg * 32 + hl];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          x[u][q] = ((const f32x4*)a.part_o)[(seg * MB + mb) * 256 + q * 64 + lane];
      }
      float M = m;
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        if (s + 4 * u <= s1) M = fmaxf(M, st[u].x);
      const float c = weight(m, M);
      l *= c;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] *= c;
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        if (s + 4 * u > s1) continue;
        const float cu = weight(st[u].x, M);
        l += st[u].y * cu;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] += x[u][i >> 2][i & 3] * cu;
      }
      m = M;
    }
  }
  {
    float* p = part + w * 18 * 64 + lane;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i * 64] = o[i];
    p[16 * 64] = m;
    p[17 * 64] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int v = 0; v < 4; ++v) M = fmaxf(M, part[(v * 18 + 16) * 64 + lane]);
  l = 0.f;
  float r[4] = {0.f, 0.f, 0.f, 0.f};  // wave w writes channels 8 w + 4 half + 0 .. 3
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float c = weight(part[(v * 18 + 16) * 64 + lane], M);
    l += part[(v * 18 + 17) * 64 + lane] * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] += part[(v * 18 + 4 * w + i) * 64 + lane] * c;
  }
  bool bad = l == 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= l == l && !finite(r[i]);
  bad = whole || (bad && node < count);
  if (__syncthreads_or(bad)) {  // (a barrier: the segments' sums in LDS are read)
    set_apart<T>(a, b, kvh, cg, mb, P, end, part);
    return;
  }
  if (node >= a.nodes) return;
  const float inv = 1.f / l;  // of a column with a row; the others are zeros
  const int64_t qrow =
      ((int64_t)b * a.nodes + node) * a.q_heads + kvh * G + (col - node * G);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] *= inv;
  write4<T>(a, qrow, 32 * mb + 8 * w + 4 * half, r, node < count);
}

constexpr int kCus = 256;

struct Kernel {
  const void* fn;
  const void* alone;  // the same with a slot per sequence, or null
  const void* join;
  int threads;
  int cols;     // columns per block
  int rows;     // rows per tile
  int width;    // DP
  int per_cu;   // blocks on a CU at a time
};

template <typename S, bool DMA>
Kernel make() {
  const void* alone = nullptr;
  if constexpr (S::WC == 16 && DMA) alone = (const void*)tree_kernel<S, DMA, true>;
  return {(const void*)tree_kernel<S, DMA, false>, alone, (const void*)tree_join<typename S::T, S::DP>,
          64 * S::NW, S::kCols, S::BK, S::DP, S::kPerCu};
}

// Few columns are bound by the rows' way from memory: 16 columns a wave, so
// that there are waves enough to hide each other's waits, and a ring of as
// many tiles as LDS holds, most of them on their way.  Many columns are
// bound by the products: 32 a wave, which halves the operand reads, and room
// for a second block, whose products run while this one forms its
// probabilities.
//
// float32: where tiles of 128 rows are fewer than CUs, tiles of 32 rows give
// more of them one (8 drafts on 508 rows, 32/8 heads of 64 / 128: 12.2 ->
// 9.3 / 13.6 -> 11.2 us; 4 x 8 on 8192 rows 31 -> 33 / 59 -> 64).
//
// 16 bits, 64 wide: tiles of 128 rows, which halves the barriers (8 x 16
// drafts on 65536 rows 223 -> 199 us, 16 x 8 on 1000 rows 16.1 -> 14.9), and
// two of them rather than four, which leaves LDS for a second block (four: 187
// and 15.4, but 128 x 8 on 264 rows 22 -> 34).  256 wide: 64 columns take 64
// rows by two waves a column rather than 32 by one (4 x 8 drafts on 32768 rows
// 63 -> 57 us); 128 columns have waves enough.  float32, 256 wide: four waves
// have the registers of eight, 32 columns 180 -> 122 us (4 x 4 drafts on 8192
// rows), 64 columns 238 -> 184 (4 x 16); 64 wide, 64 columns: room for a second
// block 62.3 -> 54-59 (4 x 16 on 8192).  More columns, 32 a wave: 4 x 64 on
// 8192 rows 148 us (64 wide), 280 (128), 314 (256, 16/2 heads): 71 to 80% of
// what a large float32 product reaches.
template <typename T>
Kernel pick(int width, int cols, bool dma, bool few) {
  if constexpr (sizeof(T) == 4) {
    if (width <= 64) {
      if (!dma) return make<Shape<T, 64, 16, 4, 2, 64, 2>, false>();
      if (cols <= 32 && few) return make<Shape<T, 64, 16, 2, 2, 32, 4>, true>();
      return cols <= 32   ? make<Shape<T, 64, 16, 2, 4, 128, 2>, true>()
             : cols <= 64 ? make<Shape<T, 64, 16, 4, 2, 64, 2>, true>()
                          : make<Shape<T, 64, 32, 4, 1, 32, 2>, true>();
    }
    if (width <= 128) {
      if (!dma) return make<Shape<T, 128, 16, 4, 2, 64, 2>, false>();
      if (cols <= 32 && few) return make<Shape<T, 128, 16, 2, 2, 32, 2>, true>();
      return cols <= 32   ? make<Shape<T, 128, 16, 2, 4, 64, 2>, true>()
             : cols <= 64 ? make<Shape<T, 128, 16, 4, 2, 64, 2>, true>()
                          : make<Shape<T, 128, 32, 4, 1, 32, 2>, true>();
    }
    if (!dma) return make<Shape<T, 256, 16, 4, 2, 32, 2>, false>();
    return cols <= 32   ? make<Shape<T, 256, 16, 2, 2, 32, 2>, true>()
           : cols <= 64 ? make<Shape<T, 256, 16, 4, 1, 32, 2>, true>()
                        : make<Shape<T, 256, 32, 4, 1, 32, 2>, true>();
  } else {
    if (width <= 64) {
      if (!dma) return make<Shape<T, 64, 16, 4, 2, 64, 2>, false>();
      return cols <= 64 ? make<Shape<T, 64, 16, 4, 2, 128, 2>, true>()
                        : make<Shape<T, 64, 32, 4, 1, 64, 2>, true>();
    }
    if (width <= 128) {
      if (!dma) return make<Shape<T, 128, 16, 4, 2, 64, 2>, false>();
      return cols <= 64 ? make<Shape<T, 128, 16, 4, 2, 64, 4>, true>()
                        : make<Shape<T, 128, 32, 4, 1, 64, 2>, true>();
    }
    if (!dma) return make<Shape<T, 256, 16, 8, 1, 32, 2>, false>();
    return cols <= 64    ? make<Shape<T, 256, 16, 4, 2, 64, 2>, true>()
           : cols <= 128 ? make<Shape<T, 256, 16, 8, 1, 32, 4>, true>()
                         : make<Shape<T, 256, 32, 4, 1, 64, 2>, true>();
  }
}

// Narrow calls run as one launch, a slot per sequence and nothing to join,
// while a sequence's K is short: the shares of the rows and the second launch
// cost 4 to 5 us, which a few tiles that follow each other do not (8 drafts,
// 32/8 heads, two launches -> one: bf16, 128 wide, 136 rows 11.4 -> 8.7 us
// and 520 rows 12.3 -> 13.6; float32, 64 wide, 136 rows 10.5 -> 8.9 and 264
// rows 10.8 -> 12.4; 256 wide, bf16 96 rows 13.9 -> 12.8 and 136 rows 14.1 ->
// 14.8, float32 32 rows 16.5 -> 13.5 and 48 rows 16.0 -> 18.4 with 16/2 heads,
// 15.6 -> 14.9 with 32/8).  Where every CU has a sequence anyway, splitting one
// gains nothing for four times as many rows (32 sequences: bf16, 128 wide, 520
// rows 22.8 -> 18.3 us); beyond that a single long sequence among short ones
// would hold the call up.
constexpr int64_t kAloneBytes = 48 * 1024;
constexpr int64_t kTilesPerSlot = 6;

struct TreePlan {
  Kernel kernel;
  int col_tiles, slots;
  bool alone;
  size_t segments, part_o, bytes;  // floats of O, bytes in all
};

TreePlan tree_plan(int batch, int nodes, int q_heads, int kv_heads, int key_dim, int value_dim,
                   int length, int dtype, bool dma, bool vec_o) {
  TreePlan p = {};
  const int width = std::max(key_dim, value_dim);
  const int cols = nodes * (q_heads / kv_heads);
  const bool few = (int64_t)batch * kv_heads * ((length + 127) / 128) < kCus;
  p.kernel = dtype == ALPX_F32   ? pick<float>(width, cols, dma, few)
             : dtype == ALPX_F16 ? pick<f16_t>(width, cols, dma, few)
                                 : pick<bf16_t>(width, cols, dma, few);
  p.col_tiles = (cols + p.kernel.cols - 1) / p.kernel.cols;
  const bool direct = vec_o && value_dim == p.kernel.width;
  // One round of blocks, every slot at least a tile; more than a block a CU
  // only where each then has several tiles, since a segment's state costs
  // about as much to write and join as two tiles (4 x 63 drafts, 32/8 heads,
  // bf16, 1000 rows: 64 wide 22.7 -> 19.1 us, 128 wide 30.2 -> 26.5; from
  // 4000 rows on nothing changes).
  const int64_t tiles = (int64_t)batch * ((length + p.kernel.rows - 1) / p.kernel.rows);
  const int64_t units = (int64_t)kv_heads * p.col_tiles;
  const int64_t share = std::min(kCus * p.kernel.per_cu / units,
                                 std::max(kCus / units, tiles / kTilesPerSlot));
  p.slots = (int)std::min(std::max<int64_t>(share, 1), tiles);
  const bool all_busy = (int64_t)batch * kv_heads * p.col_tiles >= kCus;
  p.alone = direct && p.kernel.alone &&
            (int64_t)length * p.kernel.width * (int64_t)dtype_size(dtype) <=
                (all_busy ? 4 : 1) * kAloneBytes;
  if (p.alone) {
    p.slots = batch;
    return p;
  }
  p.segments = (size_t)(p.slots + batch) * kv_heads * p.col_tiles * (p.kernel.cols / 32);
  p.part_o = p.segments * 32 * p.kernel.width;
  p.bytes = p.part_o * 4 + p.segments * 32 * sizeof(float2) + (size_t)batch * sizeof(int4);
  return p;
}

// Sums of tiles, also rounded up to whole runs of every slot, and of rows past
// the end stay in 31 bits.
bool too_many_rows(int batch, int length) {
  constexpr int64_t kSlots = kCus * 8;  // no plan has more
  return length > (1 << 30) ||
         (int64_t)batch * ((int64_t)length / 32 + 1) >= ((int64_t)1 << 31) - kSlots;
}

// Masks of every draft, and 32-bit words of them that an int counts.
bool bad_words(int words, int64_t batch_stride, int nodes) {
  return words < 0 || words >= 1 << 30 || (int64_t)words * 64 < nodes || batch_stride < 0;
}

// Blocks of the two launches; false: more threads than a grid holds.
bool tree_grids(const TreePlan& p, int batch, int kv_heads, int64_t& blocks, int64_t& joins) {
  const int64_t units = (int64_t)p.slots * kv_heads;
  blocks = (units + kXcds - 1) / kXcds * kXcds * p.col_tiles;
  joins = (int64_t)batch * kv_heads * p.col_tiles * (p.kernel.cols / 32) * (p.kernel.width / 32);
  return blocks * p.kernel.threads <= 0xffffffff && joins * 256 <= 0xffffffff;
}

bool tree_sizes_ok(int batch, int nodes, int q_heads, int kv_heads, int key_dim, int value_dim,
                   int length) {
  return batch > 0 && nodes > 0 && q_heads > 0 && kv_heads > 0 && key_dim > 0 && value_dim > 0 &&
         length > 0 && !too_many_rows(batch, length) && q_heads % kv_heads == 0 && key_dim <= 256 &&
         value_dim <= 256 &&
         (int64_t)nodes * (q_heads / kv_heads) <= (1 << 24);
}

int tree_launch(const char* what, TreeArgs a, int dtype, void* workspace, size_t workspace_bytes,
                void* stream) {
  if (!a.q || !a.k || !a.v || !a.out || !a.masks || !a.prefix)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype) || !dtype_ok(a.out_dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (a.batch <= 0 || a.nodes <= 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.key_dim <= 0 ||
      a.value_dim <= 0 || a.length <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (a.q_heads % a.kv_heads != 0)
    return fail(ALPX_EINVAL, "attention query heads must be a multiple of KV heads");
  if (a.key_dim > 256 || a.value_dim > 256)
    return fail(ALPX_EUNSUPPORTED, "%s: head widths above 256", what);
  if (!(a.scale_log2 > 0.f) || !isfinite(a.scale_log2))
    return fail(ALPX_EINVAL, "attention scale must be positive and finite");
  a.group = a.q_heads / a.kv_heads;
  const int64_t es = (int64_t)dtype_size(dtype), os = (int64_t)dtype_size(a.out_dtype);
  if ((int64_t)a.nodes * a.group > (1 << 24))
    return fail(ALPX_EUNSUPPORTED, "%s: too many drafts", what);
  if (a.ks_pos < 0 || a.ks_b < 0 || a.ks_h < 0 || a.vs_pos < 0 || a.vs_b < 0 || a.vs_h < 0)
    return fail(ALPX_EINVAL, "%s: strides must not be negative", what);
  if (too_many_rows(a.batch, a.length))
    return fail(ALPX_EUNSUPPORTED, "%s: too many rows", what);
  if (32 * std::max(a.ks_pos, a.vs_pos) * es >= ((int64_t)1 << 31))
    return fail(ALPX_EUNSUPPORTED, "%s: rows too far apart", what);
  const uintptr_t rows = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)(a.ks_pos * es) |
                         (uintptr_t)(a.ks_b * es) | (uintptr_t)(a.ks_h * es) |
                         (uintptr_t)(a.vs_pos * es) | (uintptr_t)(a.vs_b * es) |
                         (uintptr_t)(a.vs_h * es) | (uintptr_t)(a.key_dim * es) |
                         (uintptr_t)(a.value_dim * es);
  const bool dma = (rows & 15) == 0;
  a.vec_k = dma;
  a.vec_q = (((uintptr_t)a.q | (uintptr_t)(a.key_dim * es)) & 15) == 0;
  a.vec_o = a.value_dim % 4 == 0 && ((uintptr_t)a.out & (4 * os - 1)) == 0 &&
            ((uintptr_t)a.gate & (4 * es - 1)) == 0;
  // rows of values that are not finite read q and gate after others wrote out
  const int64_t cells = (int64_t)a.batch * a.nodes * a.q_heads;
  const uintptr_t out = (uintptr_t)a.out, out_end = out + (uintptr_t)(cells * a.value_dim * os);
  auto meets_out = [&](const void* x, int64_t width) {
    return x && (uintptr_t)x < out_end && out < (uintptr_t)x + (uintptr_t)(cells * width * es);
  };
  if (meets_out(a.q, a.key_dim) || meets_out(a.gate, a.value_dim))
    return fail(ALPX_EINVAL, "%s: out must not overlap q or gate", what);
  const TreePlan p = tree_plan(a.batch, a.nodes, a.q_heads, a.kv_heads, a.key_dim, a.value_dim,
                               a.length, dtype, dma, a.vec_o);
  int64_t blocks, joins;
  if (!tree_grids(p, a.batch, a.kv_heads, blocks, joins))
    return fail(ALPX_EUNSUPPORTED, "%s: too many sequences", what);
  if (((uintptr_t)workspace & 15) != 0)
    return fail(ALPX_EINVAL, "%s: workspace must be 16-byte aligned", what);
  if (workspace_bytes < p.bytes || (p.bytes > 0 && !workspace))
    return fail(ALPX_EINVAL, "%s: workspace holds %zu bytes, needs %zu", what, workspace_bytes,
                p.bytes);
  a.col_tiles = p.col_tiles;
  a.slots = p.slots;
  a.direct = a.vec_o && a.value_dim == p.kernel.width;
  a.part_o = (float*)workspace;
  a.part_st = (float2*)(a.part_o + p.part_o);
  a.found = (int4*)(a.part_st + p.segments * 32);
  hipStream_t s = (hipStream_t)stream;
  void* args[] = {&a};
  {
    TimedRegion timed(ALPX_T_DECODE, s);
    (void)hipLaunchKernel(p.alone ? p.kernel.alone : p.kernel.fn, dim3((unsigned)blocks), dim3(p.kernel.threads), args, 0, s);
  }
  if (p.alone) return check_launch(what);
  a.col_tiles = p.col_tiles * (p.kernel.cols / 32);  // groups of 32 columns
  TimedRegion timed(ALPX_T_DECODE_COMBINE, s);
  (void)hipLaunchKernel(p.kernel.join, dim3((unsigned)joins), dim3(256), args, 0, s);
  return check_launch(what);
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" size_t alpx_tree_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                            int key_dim, int value_dim, int length, int dtype) {
  if (!tree_sizes_ok(batch, nodes, q_heads, kv_heads, key_dim, value_dim, length) || !dtype_ok(dtype))
    return 0;
  size_t most = 0;  // whatever the call's alignment
  for (int i = 0; i < 4; ++i) {
    const TreePlan p = tree_plan(batch, nodes, q_heads, kv_heads, key_dim, value_dim, length, dtype,
                                 i & 1, i & 2);
    int64_t blocks, joins;
    if (tree_grids(p, batch, kv_heads, blocks, joins)) most = std::max(most, p.bytes);
  }
  return most;
}

extern "C" int alpx_tree_attention(const void* q, const void* key_cache, const void* value_cache,
                                   const uint64_t* masks, int64_t mask_batch_stride,
                                   int mask_words, const int32_t* prefix_lens,
                                   const int32_t* counts, int length, const void* gate, void* out,
                                   void* workspace, size_t workspace_bytes, int batch, int nodes,
                                   int q_heads, int kv_heads, int key_dim, int value_dim,
                                   int64_t k_pos_stride, int64_t k_batch_stride,
                                   int64_t k_head_stride, int64_t v_pos_stride,
                                   int64_t v_batch_stride, int64_t v_head_stride, float scale,
                                   int dtype, int out_dtype, void* stream) {
  if (bad_words(mask_words, mask_batch_stride, nodes))
    return fail(ALPX_EINVAL, "alpx_tree_attention: mask_words must cover every draft");
  TreeArgs a = {};
  a.q = q;
  a.k = key_cache;
  a.v = value_cache;
  a.gate = gate;
  a.out = out;
  a.masks = (const uint32_t*)masks;
  a.mask_b = 2 * mask_batch_stride;
  a.words = 2 * mask_words;
  a.prefix = prefix_lens;
  a.counts = counts;
  a.length = length;
  a.batch = batch;
  a.nodes = nodes;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.key_dim = key_dim;
  a.value_dim = value_dim;
  a.ks_pos = k_pos_stride;
  a.ks_b = k_batch_stride;
  a.ks_h = k_head_stride;
  a.vs_pos = v_pos_stride;
  a.vs_b = v_batch_stride;
  a.vs_h = v_head_stride;
  a.scale_log2 = scale * kLog2e;
  a.out_dtype = out_dtype;
  return tree_launch("alpx_tree_attention", a, dtype, workspace, workspace_bytes, stream);
}

extern "C" int alpx_tree_attention_paged(const void* q, const void* key_pages,
                                         const void* value_pages, const int32_t* block_table,
                                         int max_pages, int page_size, int num_pages,
                                         const uint64_t* masks, int64_t mask_batch_stride,
                                         int mask_words, const int32_t* prefix_lens,
                                         const int32_t* counts, int length, const void* gate,
                                         void* out, void* workspace, size_t workspace_bytes,
                                         int batch, int nodes, int q_heads, int kv_heads,
                                         int key_dim, int value_dim, float scale, int dtype,
                                         int out_dtype, void* stream) {
  if (!block_table) return fail(ALPX_EINVAL, "alpx_tree_attention_paged: null buffer");
  if (page_size < 32 || (page_size & (page_size - 1)) != 0)
    return fail(ALPX_EINVAL, "page_size must be a power of two of at least 32");
  if (max_pages <= 0 || num_pages <= 0 || kv_heads <= 0 || key_dim <= 0 || value_dim <= 0)
    return fail(ALPX_EINVAL, "alpx_tree_attention_paged: sizes must be positive");
  if (length > (int64_t)max_pages * page_size)
    return fail(ALPX_ERANGE, "attention cache length exceeds capacity");
  if (bad_words(mask_words, mask_batch_stride, nodes))
    return fail(ALPX_EINVAL, "alpx_tree_attention_paged: mask_words must cover every draft");
  TreeArgs a = {};
  a.q = q;
  a.k = key_pages;
  a.v = value_pages;
  a.gate = gate;
  a.out = out;
  a.masks = (const uint32_t*)masks;
  a.mask_b = 2 * mask_batch_stride;
  a.words = 2 * mask_words;
  a.prefix = prefix_lens;
  a.counts = counts;
  a.pages = block_table;
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.length = length;
  a.batch = batch;
  a.nodes = nodes;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.key_dim = key_dim;
  a.value_dim = value_dim;
  a.ks_pos = (int64_t)kv_heads * key_dim;
  a.ks_h = key_dim;
  a.ks_b = (int64_t)page_size * a.ks_pos;
  a.vs_pos = (int64_t)kv_heads * value_dim;
  a.vs_h = value_dim;
  a.vs_b = (int64_t)page_size * a.vs_pos;
  a.scale_log2 = scale * kLog2e;
  a.out_dtype = out_dtype;
  return tree_launch("alpx_tree_attention_paged", a, dtype, workspace, workspace_bytes, stream);
}
