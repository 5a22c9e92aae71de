// Attention of a tree of drafted tokens over a K/V cache.
//
// Sequence b holds P_b rows that every draft sees (its prefix) and, behind
// them, one row for each of its n_b drafts.  Draft i sees the prefix and
// those rows P_b + j whose bit j is set in its mask (its ancestors and
// itself, in a tree):
//   out[b, i, h] = softmax_j(scale * q[b, i, h] . K[j, h / G]) . V[j, h / G]
// over the rows it sees, times sigmoid(gate) where given; a draft that sees
// no row, and drafts at or past n_b, give zeros.
//
// The drafts of one sequence read the same rows, so a block takes columns =
// (draft, query head of one kv head) pairs, up to 128 of them, against one
// stream of K and V tiles: the cache is read once for all of them.  S^T =
// K Q^T and O^T = V^T P^T on 32 x 32 MFMA tiles: a lane owns one column
// (lane % 32), keys lie in its registers, so its mask is one word per 32
// keys, the softmax needs one exchange with the lane 32 away, and P feeds
// the second product from the registers the first one wrote.
#include <math.h>

#include <algorithm>

#include "alpx_common.h"
#include "prefill_run.h"
#include "timing.h"

namespace alpx {
namespace {

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
  float scale_log2;
  int out_dtype;
  int vec_q;          // q rows may be read, and out rows written, in vectors
};

// Loads that may come through the scalar cache: what they read is written
// by no block of the launch.
__device__ __forceinline__ int load_const(const int32_t* p) {
  return __builtin_amdgcn_readfirstlane(
      *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p);
}

// Rows of sequence b: its prefix [0, P), its drafts [P, end).
__device__ __forceinline__ void tree_rows(const TreeArgs& a, int b, int& P, int& end) {
  P = min(max(load_const(a.prefix + b), 0), a.length);
  int n = a.counts != nullptr ? load_const(a.counts + b) : a.nodes;
  n = min(max(n, 0), a.nodes);
  end = min(P + n, a.length);
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

// Shape of a kernel: T, DP (the head width rounded up to 64, 128 or 256), WK
// waves that share a column tile's keys (4 / WK waves side by side in
// columns), BK rows per K and V tile.
template <typename T, int DP_, int WK_, int BK_>
struct Shape {
  static constexpr int DP = DP_, WK = WK_, BK = BK_;
  static constexpr int WQ = 4 / WK;
  static constexpr int kCols = 32 * WQ;
  static constexpr int KR = BK / (32 * WK);      // 32-key groups per wave and tile
  static constexpr int EPU = 16 / (int)sizeof(T);  // elements per 16-byte unit
  static constexpr int U = DP / EPU;             // units per row
  static constexpr int kRowB = DP * (int)sizeof(T);
  static constexpr int kTileB = BK * kRowB;
  static constexpr int kIW = kTileB / 4096;      // direct loads per wave and tile
  static constexpr int MB = DP / 32;             // 32-channel blocks of O^T
  static_assert(BK % (32 * WK) == 0 && kIW >= 1, "tiles split evenly over the waves");
  // The rows a wave loads lie in one 32-row group of the tile, so a page of
  // 32 rows or more is looked up once per wave and tile.
  static_assert(BK / 4 <= 32 && 32 % (BK / 4) == 0, "a wave's rows share a page");
};

// Swizzles (16-byte unit u of row r is stored at u ^ swz).  K is read 32
// rows at a time, one unit each; 16-bit V by transposing reads of 8 rows,
// four units each; float V in whole 128-byte pieces of a row, any order.
template <typename S>
__device__ __forceinline__ int k_swz(int r) {
  return S::kRowB >= 256 ? (r & 15) : (r & 7);
}
template <typename T, typename S>
__device__ __forceinline__ int v_swz(int r) {
  if (sizeof(T) == 4) return 0;
  return S::kRowB >= 256 ? (((r & 7) << 1) | ((r >> 3) & 1)) : (r & 7);
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

template <typename T>
__device__ __forceinline__ bool finite(T x) {
  return fabsf(to_f32(x)) < INFINITY;
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
// then the one rounding.
template <typename T>
__device__ __forceinline__ void write4(const TreeArgs& a, int64_t row, int d0, float (&r)[4]) {
  const int n = a.value_dim - d0;
  if (n <= 0) return;
  const int64_t at = row * a.value_dim + d0;
  if (a.gate != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) r[i] *= stable_sigmoid(to_f32(((const T*)a.gate)[at + i]));
  }
  switch (a.out_dtype) {
    case ALPX_F32: store4<float>(a.out, at, r, n, a.vec_q); break;
    case ALPX_F16: store4<f16_t>(a.out, at, r, n, a.vec_q); break;
    default: store4<bf16_t>(a.out, at, r, n, a.vec_q); break;
  }
}

// One block: column tile `ct` of (sequence b, kv head).
template <typename T, int DP, int WK, int BK, bool DMA>
__global__ void __launch_bounds__(256, 1) tree_kernel(TreeArgs a) {
  typedef Shape<T, DP, WK, BK> S;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int MB = S::MB, KR = S::KR, EPU = S::EPU, U = S::U, kRowB = S::kRowB;
  constexpr int kTileB = S::kTileB;
  typedef T Unit __attribute__((ext_vector_type(EPU)));
  constexpr int NQ = DP / (2 * EPU);  // units of a query row per lane (half of them)
  constexpr int kMergeB = (WK - 1) * S::WQ * (MB * 16 + 2) * 256;
  constexpr int kLds = 4 * kTileB > kMergeB ? 4 * kTileB : kMergeB;
  __shared__ __attribute__((aligned(1024))) char smem[kLds];  // K 0, V 0, K 1, V 1

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave % S::WQ, wk = wave / S::WQ;
  const int hl = lane & 31, half = lane >> 5;

  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds;
  const int ct = at % a.col_tiles;
  const int unit = (at / a.col_tiles) * kXcds + xcd;
  if (unit >= a.batch * a.kv_heads) return;
  const int b = unit / a.kv_heads, kvh = unit % a.kv_heads;
  int P, end;
  tree_rows(a, b, P, end);
  const int count = end - P;

  const int G = a.group;
  const int col = ct * S::kCols + 32 * wq + hl;
  const int node = col / G;
  const bool in_range = node < a.nodes, live = node < count;
  const int64_t qrow = ((int64_t)b * a.nodes + (in_range ? node : 0)) * a.q_heads +
                       kvh * G + (col - node * G);
  const uint32_t* mask = a.masks + b * a.mask_b + (int64_t)(in_range ? node : 0) * a.words;

  // B operand of S^T: this lane's units of its column's query row (unit
  // 2 j + half of every pair j), zero past the head width.
  Unit qv[NQ];
  {
    const T* qp = (const T*)a.q + qrow * a.key_dim;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int d = EPU * (2 * j + half);
      Unit x = {};
      if (live) {
        if (a.vec_q && d + EPU <= a.key_dim) {
          x = *(const Unit*)(qp + d);
        } else {
#pragma unroll
          for (int e = 0; e < EPU; ++e)
            if (d + e < a.key_dim) x[e] = qp[d + e];
        }
      }
      qv[j] = x;
    }
  }

  f32x16 o[MB];  // O^T[channel 32 mb + 8 (r / 4) + 4 half + r % 4][column]
  float m, l;    // the column's reference score and this lane's share of the sum of P

  // Rows [start, stop) in tiles of BK.
  const int start = 0, stop = end;
  const int nt = (stop - start + BK - 1) / BK;

  // Tile loads: wave w fills rows [w BK / 4, (w + 1) BK / 4) of a tile, all
  // in its 32-row group `grp`.
  constexpr int kRows = BK / 4;
  const int grp = wave * kRows / 32 * 32;
  uint32_t kofs[S::kIW], vofs[S::kIW];
#pragma unroll
  for (int i = 0; i < S::kIW; ++i) {
    const int sl = (wave * S::kIW + i) * 64 + lane;
    const int r = sl / U;
    const int uk = (sl % U) ^ k_swz<S>(r), uv = (sl % U) ^ v_swz<T, S>(r);
    // units past the head width: an offset past every row, which reads zero
    kofs[i] = uk * EPU < a.key_dim
                  ? (uint32_t)(((int64_t)(r - grp) * a.ks_pos + EPU * uk) * (int64_t)sizeof(T))
                  : 0x80000000u;
    vofs[i] = uv * EPU < a.value_dim
                  ? (uint32_t)(((int64_t)(r - grp) * a.vs_pos + EPU * uv) * (int64_t)sizeof(T))
                  : 0x80000000u;
  }
  const uint32_t lbase = (uint32_t)(uintptr_t)(lds_void_t*)smem;

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
  auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
    const int row0 = start + t * BK + grp;
    const int rows = __builtin_amdgcn_readfirstlane(min(max(stop - row0, 0), 32));
    const T *kb = (const T*)a.k, *vb = (const T*)a.v;
    if (rows > 0) group_base(row0, kb, vb);
    if constexpr (DMA) {
      const i32x4 rk = rsrc_words((uint64_t)(uintptr_t)kb,
                                  (uint32_t)(rows * a.ks_pos * (int64_t)sizeof(T)));
      const i32x4 rv = rsrc_words((uint64_t)(uintptr_t)vb,
                                  (uint32_t)(rows * a.vs_pos * (int64_t)sizeof(T)));
      const uint32_t dst = lbase + buf * 2 * kTileB + wave * S::kIW * 1024;
#pragma unroll
      for (int i = 0; i < S::kIW; ++i) lds_dma16(rk, dst + i * 1024, kofs[i]);
#pragma unroll
      for (int i = 0; i < S::kIW; ++i) lds_dma16(rv, dst + kTileB + i * 1024, vofs[i]);
    } else {
      // any head width, stride or alignment: element by element
      T* dst = (T*)(smem + buf * 2 * kTileB);
      for (int i = lane; i < kRows * DP; i += 64) {
        const int r = wave * kRows + i / DP, d = i % DP;
        const bool in = r - grp < rows;
        const T kx = in && d < a.key_dim ? kb[(int64_t)(r - grp) * a.ks_pos + d] : from_f32<T>(0.f);
        const T vx = in && d < a.value_dim ? vb[(int64_t)(r - grp) * a.vs_pos + d] : from_f32<T>(0.f);
        const int u = d / EPU, e = d % EPU;
        dst[r * DP + (u ^ k_swz<S>(r)) * EPU + e] = kx;
        dst[kTileB / (int)sizeof(T) + r * DP + (u ^ v_swz<T, S>(r)) * EPU + e] = vx;
      }
    }
  };

  // One pass over the rows.  SAFE: a row that one column sees and another
  // does not may hold an infinity or a NaN, and 0 times it is no 0: the
  // product takes the finite values alone, and each column adds the others
  // of the rows that it sees.
  auto walk = [&](auto safe_) __attribute__((always_inline)) {
    constexpr bool SAFE = decltype(safe_)::value;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[mb][r] = 0.f;
    if (nt > 0) load_tile(0, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
      const int buf = t & 1;
      if (t + 1 < nt) load_tile(t + 1, buf ^ 1);
      const char* kt = smem + buf * 2 * kTileB;
      const char* vt = kt + kTileB;
#pragma unroll
      for (int kr = 0; kr < KR; ++kr) {
        const int g0 = 32 * (wk * KR + kr);       // this wave's keys of the tile
        const int key0 = start + t * BK + g0;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
        const int row = g0 + hl;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          const Unit ka = *(const Unit*)(kt + row * kRowB + ((2 * j + half) ^ k_swz<S>(row)) * 16);
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s = mfma32x32x2(ka[e], qv[j][e], s);
          } else {
            s = mfma32x32x16(ka, qv[j], s);
          }
        }
        uint32_t bits = 0xffffffffu;
        if (SAFE || key0 + 32 > P) {  // not all of these keys are prefix rows
          bits = seen_bits(mask, a.words, P, stop, key0, live);
          const uint32_t mine = bits >> (4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(mine & (1u << (8 * (r >> 2) + (r & 3))))) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx *= a.scale_log2;
        // the reference moves only when a score exceeds it by more than
        // kRescale, so P <= 2^kRescale and the sums keep their range
        if (__ballot(mx > m + kRescale) != 0) {
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          if (mx > m + kRescale) {
            const float c = fast_exp2(m - mx);  // 0 while m is -inf
            l *= c;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (!SAFE || finite(o[mb][r])) o[mb][r] *= c;
            m = mx;
          }
        }
        const float off = m == -INFINITY ? 0.f : m;
        float ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = fast_exp2(fmaf(s[r], a.scale_log2, -off));
          ps += s[r];
        }
        l += ps;
        // O^T += V^T P^T.  Any order of the keys will do as long as both
        // operands have the same: slot e of lane half h is key 16 ks +
        // 8 (e / 4) + 4 h + e % 4, which is where P already lies.
        bool bad = false;
        if constexpr (F32) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int vr = g0 + 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
              float x = *(const float*)(vt + vr * kRowB + 128 * mb + 4 * hl);
              if (SAFE && !finite(x)) {
                bad = true;
                x = 0.f;
              }
              o[mb] = mfma32x32x2(x, s[r], o[mb]);
            }
          }
        } else {
          typedef typename Vec8<T>::type V8;
          typedef typename Vec4<T>::type V4;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            V8 p;
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = from_f32<T>(s[8 * ks + e]);
            // transposing reads: lane 4 k + q of 16 supplies row k, channels
            // 4 q .. 4 q + 3, and receives channel lane % 16 of the four rows
            const int vr = g0 + 16 * ks + 4 * half + ((lane & 15) >> 2);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
              const int u = 4 * mb + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
              const T* p0 = (const T*)(vt + vr * kRowB + (u ^ v_swz<T, S>(vr)) * 16 + 8 * (lane & 1));
              const T* p1 = (const T*)(vt + (vr + 8) * kRowB + (u ^ v_swz<T, S>(vr + 8)) * 16 +
                                       8 * (lane & 1));
              const V4 x0 = lds_read_tr4(p0), x1 = lds_read_tr4(p1);
              V8 x = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
              if constexpr (SAFE) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (!finite(x[e])) {
                    bad = true;
                    x[e] = from_f32<T>(0.f);
                  }
              }
              o[mb] = mfma32x32x16(x, p, o[mb]);
            }
          }
        }
        if constexpr (SAFE) {
          if (__ballot(bad) != 0) {
#pragma clang loop unroll(disable)
            for (int key = 0; key < 32; ++key) {
              if (!(bits >> key & 1u)) continue;
              const int vr = g0 + key;
#pragma unroll
              for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const int d = 32 * mb + 8 * (r >> 2) + 4 * half + (r & 3);
                  const T x = *(const T*)(vt + vr * kRowB + ((d / EPU) ^ v_swz<T, S>(vr)) * 16 +
                                          (d % EPU) * (int)sizeof(T));
                  if (!finite(x)) o[mb][r] += to_f32(x);
                }
            }
          }
        }
      }
      __builtin_amdgcn_s_waitcnt(0);  // the next tile is in LDS
      __syncthreads();
    }
  };

  walk(std::false_type());
  bool bad = false;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= !(fabsf(o[mb][r]) < INFINITY);
  if (__syncthreads_or(bad)) walk(std::true_type());

  l += __shfl_xor(l, 32);
  if constexpr (WK > 1) {
    // the waves of a column tile's keys, joined in LDS by the first of them
    constexpr int kPart = (MB * 16 + 2) * 64;  // floats per wave
    float* part = (float*)smem;
    if (wk > 0) {
      float* p = part + ((wk - 1) * S::WQ + wq) * kPart + lane;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) p[(mb * 16 + r) * 64] = o[mb][r];
      p[MB * 16 * 64] = m;
      p[(MB * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int w = 0; w < WK - 1; ++w) {
      const float* p = part + (w * S::WQ + wq) * kPart + lane;
      const float m1 = p[MB * 16 * 64], l1 = p[(MB * 16 + 1) * 64];
      const float M = fmaxf(m, m1);
      // a part that saw no row has l = 0 and O = 0; one that saw a NaN keeps it
      const float c0 = m == -INFINITY ? 1.f : fast_exp2(m - M);
      const float c1 = m1 == -INFINITY ? 1.f : fast_exp2(m1 - M);
      l = l * c0 + l1 * c1;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x0 = o[mb][r], x1 = p[(mb * 16 + r) * 64];
          o[mb][r] = (finite(x0) ? x0 * c0 : x0) + (finite(x1) ? x1 * c1 : x1);
        }
      m = M;
    }
  }
  if (!in_range) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = live ? o[mb][4 * q + i] * inv : 0.f;
      write4<T>(a, qrow, 32 * mb + 8 * q + 4 * half, r);
    }
}

struct Kernel {
  const void* fn;
  int cols;  // columns per block
};

template <typename T, int DP, int WK, int BK, bool DMA>
Kernel make() {
  return {(const void*)tree_kernel<T, DP, WK, BK, DMA>, Shape<T, DP, WK, BK>::kCols};
}

template <typename T>
Kernel pick(int width, bool dma) {
  constexpr int B64 = sizeof(T) == 4 ? 32 : 64;
  if (width <= 64) return dma ? make<T, 64, 1, B64, true>() : make<T, 64, 1, B64, false>();
  if (width <= 128) return dma ? make<T, 128, 1, B64, true>() : make<T, 128, 1, B64, false>();
  return dma ? make<T, 256, 1, 32, true>() : make<T, 256, 1, 32, false>();
}

int tree_launch(const char* what, TreeArgs a, int dtype, void* workspace, size_t workspace_bytes,
                void* stream) {
  (void)workspace;
  (void)workspace_bytes;
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
  if (32 * std::max(a.ks_pos, a.vs_pos) * es >= ((int64_t)1 << 31))
    return fail(ALPX_EUNSUPPORTED, "%s: rows too far apart", what);
  const uintptr_t rows = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)(a.ks_pos * es) |
                         (uintptr_t)(a.ks_b * es) | (uintptr_t)(a.ks_h * es) |
                         (uintptr_t)(a.vs_pos * es) | (uintptr_t)(a.vs_b * es) |
                         (uintptr_t)(a.vs_h * es) | (uintptr_t)(a.key_dim * es) |
                         (uintptr_t)(a.value_dim * es);
  const bool dma = (rows & 15) == 0;
  a.vec_q = (((uintptr_t)a.q | (uintptr_t)(a.key_dim * es)) & 15) == 0 &&
            (((uintptr_t)a.out | (uintptr_t)(a.value_dim * os)) & (4 * os - 1)) == 0;
  const int width = std::max(a.key_dim, a.value_dim);
  const Kernel kernel = dtype == ALPX_F32   ? pick<float>(width, dma)
                        : dtype == ALPX_F16 ? pick<f16_t>(width, dma)
                                            : pick<bf16_t>(width, dma);
  a.col_tiles = (a.nodes * a.group + kernel.cols - 1) / kernel.cols;
  const int64_t units = (int64_t)a.batch * a.kv_heads;
  const int64_t blocks = (units + kXcds - 1) / kXcds * kXcds * a.col_tiles;
  if (blocks > 0x7fffffff) return fail(ALPX_EUNSUPPORTED, "%s: too many sequences", what);
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_DECODE, s);
  void* args[] = {&a};
  if (hipLaunchKernel(kernel.fn, dim3((unsigned)blocks), dim3(256), args, 0, s) != hipSuccess) {
    return check_launch(what);
  }
  return check_launch(what);
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" size_t alpx_tree_workspace_bytes(int, int, int, int, int, int, int, int) { return 0; }

extern "C" int alpx_tree_attention(const void* q, const void* key_cache, const void* value_cache,
                                   const uint64_t* masks, int64_t mask_batch_stride,
                                   int mask_words, const int32_t* prefix_lens,
                                   const int32_t* counts, int length, const void* gate, void* out,
                                   void* workspace, size_t workspace_bytes, int batch, int nodes, int q_heads, int kv_heads, int key_dim,
                                   int value_dim, int64_t k_pos_stride, int64_t k_batch_stride,
                                   int64_t k_head_stride, int64_t v_pos_stride,
                                   int64_t v_batch_stride, int64_t v_head_stride, float scale,
                                   int dtype, int out_dtype, void* stream) {
  if (mask_words < 0 || (int64_t)mask_words * 64 < nodes || mask_batch_stride < 0)
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
  if (mask_words < 0 || (int64_t)mask_words * 64 < nodes || mask_batch_stride < 0)
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
