// Packed tokens of any sequences and positions on their way into a page pool:
// queries and keys turned by their positions, keys and values written to
// their rows, as they are or as 4-bit codes; and rows of codes read back.
//
//   theta_p = position * scale * base^(-2 p / (2 R)), p < R
//   (a, b) -> (a cos - b sin, a sin + b cos)
// of channels (2 p, 2 p + 1) ("norm") or (p, p + R) ("neox"); channels from
// 2 R on stay.  A group of 32 channels of a 4-bit row is stored as
//   least = f16(min), step = f16((max - least) / 15),
//   code = clamp(round((x - least) / step), 0, 15), 0 where the step is 0,
// in float64, rounded through float32: where a code, a step or a least value
// changes must not depend on the order of operations.
#include <math.h>

#include <algorithm>

#include "alpx_common.h"
#include "q4_internal.h"
#include "rope_internal.h"
#include "timing.h"

namespace alpx {
namespace {

constexpr int kThreads = 256;
// Items of a thread of q4_rows_kernel, 32 bytes of output: 8192 rows of 8 heads of
// 128 to bf16 12.5 us with one, 11.6 with two and four; 4133 rows to float32 with
// one 0.4 us less than with two.
template <typename T>
constexpr int kFlight = sizeof(T) == 4 ? 1 : 2;

constexpr double kMostFrequency = 4.0;  // radians a position: what angle_of covers

struct RotaryArgs {
  const void* q;     // [T, Hq, D]
  const void* k;     // [T, Hkv, D]
  const void* v;     // [T, Hkv, Dv]
  void* q_out;       // [T, Hq, D]
  void* kc;          // [rows, Hkv, D], or codes
  void* vc;          // [rows, Hkv, Dv], or codes
  f16_t* ks;         // scales, for codes
  f16_t* vs;
  const int32_t* slots;      // [T], rows of the pool; others write no row
  const int32_t* positions;  // [T]; unused with R = 0
  int64_t rows;
  int Hq, Hkv, D, Dv, R, page_shift;
  bool neox;
  bool vec;   // rows may be read and written in vectors of 8 channels
  bool pvec;  // and the partners of a neox rotation too
  double inv[kMaxPairs];
};

// sin and cos of a theta below 2^33 in size, to some 2^-52 of 1: what whole quarter
// turns leave (an fma by each of the two parts of pi / 2 loses nothing that
// counts), then the powers up to where the next one is below 2^-60 at pi / 4.
__device__ __forceinline__ double2 angle_of(double theta) {
  constexpr double kQuarter = 1.570796326794896558, kRest = 6.123233995736766e-17;
  const double n = rint(theta * 0.63661977236758134);
  const double x = fma(-n, kRest, fma(-n, kQuarter, theta)), z = x * x;
  constexpr double kSin[8] = {-1.0 / 6,          1.0 / 120,           -1.0 / 5040,
                              1.0 / 362880,      -1.0 / 39916800,     1.0 / 6227020800.0,
                              -1.0 / 1307674368000.0, 1.0 / 355687428096000.0};
  constexpr double kCos[8] = {-1.0 / 2,          1.0 / 24,            -1.0 / 720,
                              1.0 / 40320,       -1.0 / 3628800,      1.0 / 479001600,
                              -1.0 / 87178291200.0, 1.0 / 20922789888000.0};
  double s = kSin[7], c = kCos[7];
#pragma unroll
  for (int i = 6; i >= 0; --i) {
    s = fma(s, z, kSin[i]);
    c = fma(c, z, kCos[i]);
  }
  s = fma(s * z, x, x);
  c = fma(c, z, 1.0);
  const int turns = (int)(int64_t)n & 3;
  const double ys = turns & 1 ? c : s, yc = turns & 1 ? s : c;
  return make_double2(turns == 1 || turns == 2 ? -yc : yc, turns >= 2 ? -ys : ys);
}

template <typename T>
struct Row8 {
  T x[8];
};
template <typename T>
__device__ __forceinline__ Row8<T> load8(const T* p, int n, bool vec) {
  Row8<T> r = {};
  if (vec) {
    constexpr int kVecs = sizeof(T) * 8 / 16;
    u32x4 w[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) w[i] = ((const u32x4*)p)[i];
    __builtin_memcpy(&r, w, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) r.x[i] = p[i];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Row8<T>& r, int n, bool vec) {
  if (vec) {
    constexpr int kVecs = sizeof(T) * 8 / 16;
    u32x4 w[kVecs];
    __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < kVecs; ++i) ((u32x4*)p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = r.x[i];
  }
}

// The 8 channels from c0 of a row turned by its token's angles, in A (float,
// or double where the result is coded).
template <typename A, typename T, typename Angle>
__device__ __forceinline__ void turn8(const RotaryArgs& a, const T* row, int c0, int n,
                                      const Row8<T>& raw, const Angle* cs, A (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (A)to_f32(raw.x[i]);
  if (c0 >= 2 * a.R) return;
  if (!a.neox) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (c0 + i >= 2 * a.R) continue;
      const Angle r = cs[(c0 + i) >> 1];
      const A lo = y[i], hi = y[i + 1];
      y[i] = lo * r.x - hi * r.y;
      y[i + 1] = lo * r.y + hi * r.x;
    }
    return;
  }
  Row8<T> far = {};
  if (a.pvec) {  // all eight lie in one half
    far = load8(row + (c0 < a.R ? c0 + a.R : c0 - a.R), 8, true);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i;
      if (i < n && c < 2 * a.R) far.x[i] = row[c < a.R ? c + a.R : c - a.R];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = c0 + i;
    if (c >= 2 * a.R) continue;
    const bool first = c < a.R;
    const Angle r = cs[first ? c : c - a.R];
    const A p = (A)to_f32(far.x[i]);
    y[i] = first ? y[i] * r.x - p * r.y : p * r.y + y[i] * r.x;
  }
}

// One token per grid row, eight channels per thread; grid y shares out a
// token's rows (queries, keys, values, in this order).  Bound by memory: 4133
// tokens of 32 + 8 + 8 heads of 128, bf16, 101.6 MB in 19.2 us (5.3 TB/s).
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_rows_kernel(RotaryArgs a) {
  __shared__ float2 cs[kMaxPairs];
  const int t = blockIdx.x;
  const int slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.rows;
  const int per = (a.D + 7) >> 3, per_v = (a.Dv + 7) >> 3;
  const int turned = (a.Hq + a.Hkv) * per, items = turned + a.Hkv * per_v;
  for (int p = threadIdx.x; p < a.R; p += kThreads) {
    const double2 r = angle_of((double)a.positions[t] * a.inv[p]);
    cs[p] = make_float2((float)r.x, (float)r.y);
  }
  __syncthreads();
  for (int j = blockIdx.y * kThreads + threadIdx.x; j < items; j += kThreads * gridDim.y) {
    if (j >= turned) {
      if (!stored) return;
      const int h = (j - turned) / per_v, c0 = 8 * ((j - turned) - h * per_v);
      const int n = min(8, a.Dv - c0);
      const Row8<T> r = load8((const T*)a.v + ((int64_t)t * a.Hkv + h) * a.Dv + c0, n, a.vec);
      store8((T*)a.vc + ((int64_t)slot * a.Hkv + h) * a.Dv + c0, r, n, a.vec);
      continue;
    }
    const int row = j / per, c0 = 8 * (j - row * per), n = min(8, a.D - c0);
    const bool is_q = row < a.Hq;
    if (!is_q && !stored) continue;
    const int h = is_q ? row : row - a.Hq;
    const T* src = is_q ? (const T*)a.q + ((int64_t)t * a.Hq + h) * a.D
                        : (const T*)a.k + ((int64_t)t * a.Hkv + h) * a.D;
    float y[8];
    turn8(a, src, c0, n, load8(src + c0, n, a.vec), cs, y);
    Row8<T> out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.x[i] = from_f32<T>(y[i]);
    T* dst = is_q ? (T*)a.q_out + ((int64_t)t * a.Hq + h) * a.D
                  : (T*)a.kc + ((int64_t)slot * a.Hkv + h) * a.D;
    store8(dst + c0, out, n, a.vec);
  }
}

// Over the four neighbouring threads of a group (whole rows of threads are in
// step here, so their lanes are).
template <int CTRL>
__device__ __forceinline__ float quad(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ double quad(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kQuad1 = 0xb1, kQuad2 = 0x4e;  // lane ^ 1, lane ^ 2
template <typename A, typename F>
__device__ __forceinline__ A over_group(A x, F f) {
  x = f(x, quad<kQuad1>(x));
  return f(x, quad<kQuad2>(x));
}
__device__ __forceinline__ float least_of(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double least_of(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float most_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most_of(double a, double b) { return fmax(a, b); }

// Through float32, in two roundings: left to itself the compiler makes one
// (and a long one) of them.
__device__ __forceinline__ f16_t to_half(double x) {
  float y = (float)x;
  asm("" : "+v"(y));
  return (f16_t)y;
}

// The codes of 8 channels, and the step and least value of the group of four
// neighbouring threads that share them.  A: double, or float where the
// channels are values of 32 bits or fewer as they stand.
template <typename A>
__device__ __forceinline__ uint32_t codes8(const A (&x)[8], f16_t& step, f16_t& least) {
  A lo = x[0], hi = x[0], odd = x[0] * (A)0;  // odd: NaN where a channel is not finite
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = least_of(lo, x[i]);
    hi = most_of(hi, x[i]);
    odd += x[i] * (A)0;
  }
  lo = over_group(lo, [](A a, A b) { return least_of(a, b); });
  hi = over_group(hi, [](A a, A b) { return most_of(a, b); });
  odd = over_group(odd, [](A a, A b) { return a + b; });
  constexpr double kMost = 65504.0;
  least = to_half(fmin(fmax((double)lo, -kMost), kMost));
  // a fifteenth, rounded as a division rounds: the quotient by the rounded
  // reciprocal, set right by what it leaves
  constexpr double kFifteenth = 1.0 / 15.0;
  const double range = (double)hi - (double)least;
  double fifteenth = range * kFifteenth;
  fifteenth = fma(fma(-15.0, fifteenth, range), kFifteenth, fifteenth);
  step = to_half(fmin(fmax(fifteenth, 0.0), kMost));
  if (odd != odd) {  // the whole group reads as NaN
    least = (f16_t)__builtin_nanf("");
    step = (f16_t)0.f;
  }
  const float d = (float)step;
  if (!(d > 0.f)) return 0u;
  const A m = (A)(float)least;
  const float inv = __builtin_amdgcn_rcpf(d);
  // Adding 2^23 rounds to whole numbers and leaves them in the low bits; the
  // bits of 2^23 itself, shifted along, are taken off the word beforehand.
  // The float quotient is some 1e-5 off at most (16 2^-24 for the difference,
  // the product and the reciprocal each): nearer than 1e-4 to a border the
  // exact one decides.
  constexpr float kWhole = 8388608.f;
  uint32_t word = 0u - 0xfb000000u;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf((float)(x[i] - m) * inv, 0.f), 15.f);
    const float y = c + kWhole;
    far = fmaxf(far, fabsf(c - (y - kWhole)));
    word += __builtin_bit_cast(uint32_t, y) << (4 * i);
  }
  if (far > 0.4999f) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double c = rint(((double)x[i] - (double)(float)least) / (double)d);
      word |= (uint32_t)fmin(fmax(c, 0.0), 15.0) << (4 * i);
    }
  }
  return word;
}

// The same with the pool's rows as codes.  A thread keeps its channels and
// goes down the rows: queries, then keys and values, from the last block on
// where blocks share a token.  Keys are turned and coded in float64 (where a
// code changes must not depend on the order of operations), values coded in
// float32, which holds them.  4133 tokens of 16 + 2 + 2 heads of 256, 64
// channels turned, bf16: 79 MB in 22.9 us (3.4 TB/s); without the coding 21.1,
// without the angles 21.8, queries alone 16.6: seven waves a SIMD do not cover
// what a row waits for, and two rows at a time (78 registers) take as long.
template <typename T>
__global__ void __launch_bounds__(kThreads) q4_append_kernel(RotaryArgs a) {
  __shared__ double2 cs[kMaxPairs];
  __shared__ float2 csf[kMaxPairs];
  const int t = blockIdx.x;
  const int slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.rows;
  const int per = a.D >> 3, groups = a.D / kQ4Group, size = 1 << a.page_shift;
  const int down = kThreads / per, first = threadIdx.x / per;
  const int o = threadIdx.x - first * per, c0 = 8 * o;
  const bool works = first < down;
  const int q_rows = works ? a.Hq : 0, kv_rows = works && stored ? 2 * a.Hkv : 0;
  const int stride = down * gridDim.y, row0 = blockIdx.y * down + first;
  const int kv_row0 = (gridDim.y - 1 - blockIdx.y) * down + first;
  for (int p = threadIdx.x; p < a.R; p += kThreads) {
    const double2 r = angle_of((double)a.positions[t] * a.inv[p]);
    cs[p] = r;
    csf[p] = make_float2((float)r.x, (float)r.y);
  }
  __syncthreads();
  for (int row = row0; row < q_rows; row += stride) {
    const int64_t at = ((int64_t)t * a.Hq + row) * a.D;
    const T* src = (const T*)a.q + at;
    int at0 = c0;  // (or a row's angles stay in registers: 92 of them, 31 us for 28)
    asm volatile("" : "+v"(at0));
    float y[8];
    turn8(a, src, at0, 8, load8(src + c0, 8, a.vec), csf, y);
    Row8<T> out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.x[i] = from_f32<T>(y[i]);
    store8((T*)a.q_out + at + c0, out, 8, a.vec);
  }
  for (int row = kv_row0; row < kv_rows; row += stride) {
    const bool is_k = row < a.Hkv;
    const int h = is_k ? row : row - a.Hkv;
    const T* src = (const T*)(is_k ? a.k : a.v) + ((int64_t)t * a.Hkv + h) * a.D;
    const Row8<T> raw = load8(src + c0, 8, a.vec);
    f16_t step, least;
    uint32_t word;
    if (is_k) {
      int at0 = c0;
      asm volatile("" : "+v"(at0));
      double y[8];
      turn8(a, src, at0, 8, raw, cs, y);
      word = codes8(y, step, least);
    } else {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = to_f32(raw.x[i]);
      word = codes8(y, step, least);
    }
    const int64_t head = (int64_t)(slot >> a.page_shift) * a.Hkv + h;
    const int r = slot & (size - 1), g = o >> 2;
    ((uint32_t*)(is_k ? a.kc : a.vc))[(head * size + r) * per + o] = word;
    if ((o & 3) == 0) {
      f16_t* s = (is_k ? a.ks : a.vs) + (head * 2 * groups + g) * size + r;
      s[0] = step;
      s[(int64_t)groups * size] = least;
    }
  }
}

struct Q4RowsArgs {
  const uint32_t* codes[2];  // K, V
  const f16_t* scales[2];
  void* out[2];              // [T, Hkv, D]
  const int32_t* slots;      // [T]
  int64_t rows, items;       // rows of the pool; 8-channel items of one of K, V
  int Hkv, D, page_shift;
};

// Eight channels of kFlight rows per thread, whose loads are on their way
// together; grid y: K, V.  Bound by memory, above all by its writes: 33.5 MB of
// them and 10.5 MB of codes and scales in 11.6 us (3.8 TB/s).
template <typename T>
__global__ void __launch_bounds__(kThreads) q4_rows_kernel(Q4RowsArgs a) {
  constexpr int kFlight = alpx::kFlight<T>, kSpan = kFlight * kThreads;  // items of a block
  const int per = a.D >> 3, groups = a.D / kQ4Group, size = 1 << a.page_shift;
  const int which = blockIdx.y;
  const uint32_t* codes = which ? a.codes[1] : a.codes[0];
  const f16_t* scales = which ? a.scales[1] : a.scales[0];
  T* dst = (T*)(which ? a.out[1] : a.out[0]);
  // one long division per block; from there on small ones
  const int magic = (65536 + per - 1) / per;  // n / per = n magic >> 16 for n below 2048
  const float inv = 1.f / (float)a.Hkv;
  for (int64_t j0 = (int64_t)blockIdx.x * kSpan; j0 < a.items; j0 += (int64_t)gridDim.x * kSpan) {
    const int64_t row0 = j0 / per, t0 = row0 / a.Hkv;
    const int o0 = (int)(j0 - row0 * per), h0 = (int)(row0 - t0 * a.Hkv);
    int slot[kFlight], h[kFlight], o[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int n = o0 + u * kThreads + (int)threadIdx.x, down = n * magic >> 16;
      o[u] = n - down * per;
      h[u] = h0 + down;
      const int ahead = a.Hkv > kSpan ? (h[u] >= a.Hkv) : (int)(((float)h[u] + 0.5f) * inv);
      h[u] -= ahead * a.Hkv;
      slot[u] = j0 + u * kThreads + threadIdx.x < a.items ? a.slots[t0 + ahead] : -1;
    }
    uint32_t word[kFlight];
    f16_t step[kFlight], least[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const bool in = slot[u] >= 0 && slot[u] < a.rows;
      const int at = in ? slot[u] : 0;
      const int64_t head = (int64_t)(at >> a.page_shift) * a.Hkv + h[u];
      const int r = at & (size - 1);
      const f16_t* s = scales + (head * 2 * groups + o[u] / 4) * size + r;
      word[u] = codes[(head * size + r) * per + o[u]];
      step[u] = s[0];
      least[u] = s[(int64_t)groups * size];
      if (!in) {
        word[u] = 0;
        step[u] = least[u] = (f16_t)0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int64_t j = j0 + u * kThreads + threadIdx.x;
      if (j >= a.items) break;
      Row8<T> out;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        out.x[i] = from_f32<T>(fmaf((float)((word[u] >> (4 * i)) & 15u), (float)step[u], (float)least[u]));
      store8(dst + 8 * j, out, 8, true);
    }
  }
}

// The host's part that both forms of the append share; 0 or a status.
int rotary_args(const char* what, RotaryArgs& a, const void* query, const void* key,
                const void* value, void* query_out, void* key_rows, void* value_rows,
                const int32_t* slots, const int32_t* positions, int dtype, int tokens, int q_heads,
                int kv_heads, int head_dim, int value_dim, int rotary_dim, int style, double base,
                double scale) {
  if (!key || !value || !key_rows || !value_rows || !slots || (q_heads > 0 && (!query || !query_out)) ||
      (rotary_dim > 0 && !positions))
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (tokens <= 0 || q_heads < 0 || kv_heads <= 0 || head_dim <= 0 || value_dim <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (head_dim > kRopeMaxDim || value_dim > kRopeMaxDim)
    return fail(ALPX_EUNSUPPORTED, "%s: head dims above %d", what, kRopeMaxDim);
  if (((int64_t)q_heads + 2 * (int64_t)kv_heads) * ((std::max(head_dim, value_dim) + 7) / 8) >
      0x7fffffff - 2 * kThreads * 1024)
    return fail(ALPX_EUNSUPPORTED, "%s: too many heads", what);
  if ((int64_t)tokens * kThreads > 0xffffffff)  // a block a token: the threads of a launch
    return fail(ALPX_EUNSUPPORTED, "%s: too many tokens", what);
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(ALPX_EINVAL, "%s: rotary_dim must be even and at most the head width", what);
  if (style != ALPX_ROTARY_NORM && style != ALPX_ROTARY_NEOX)
    return fail(ALPX_EINVAL, "%s: unknown rotary style", what);
  if (rotary_dim > 0 && (!(base > 0.0) || !isfinite(base) || !(scale > 0.0) || !isfinite(scale)))
    return fail(ALPX_EINVAL, "%s: frequency base and scale must be positive and finite", what);
  const int64_t es = (int64_t)dtype_size(dtype), row = tokens * (int64_t)head_dim * es;
  const int64_t turned = q_heads > 0 ? q_heads * row : 0;
  if (q_heads == 0) query = query_out = nullptr;
  if (meet(query_out, turned, query, turned) || meet(query_out, turned, key, kv_heads * row) ||
      meet(query_out, turned, value, tokens * (int64_t)kv_heads * value_dim * es))
    return fail(ALPX_EINVAL, "%s: query_out must not overlap an input", what);
  a.q = query;
  a.k = key;
  a.v = value;
  a.q_out = query_out;
  a.kc = key_rows;
  a.vc = value_rows;
  a.slots = slots;
  a.positions = positions;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.Dv = value_dim;
  a.R = rotary_dim / 2;
  a.neox = style == ALPX_ROTARY_NEOX;
  if (a.R > 0) {
    // (64 powers take a few microseconds, more than the rest of a call)
    static thread_local struct {
      double base, scale;
      int R;
      double inv[kMaxPairs];
    } last = {};
    if (last.R != a.R || last.base != base || last.scale != scale) {
      inverse_frequencies(last.inv, a.R, base, scale);
      last.R = a.R;
      last.base = base;
      last.scale = scale;
    }
    // (rising with a base below 1; positions below 2^31 make angles below 2^33)
    if (!(std::max(last.inv[0], last.inv[a.R - 1]) <= kMostFrequency))
      return fail(ALPX_EUNSUPPORTED, "%s: frequencies above 4", what);
    std::copy(last.inv, last.inv + a.R, a.inv);
  }
  return ALPX_OK;
}

// Few tokens: a token's rows are shared out over blocks.
dim3 rotary_grid(const RotaryArgs& a, int tokens) {
  const int items = (a.Hq + a.Hkv) * ((a.D + 7) / 8) + a.Hkv * ((a.Dv + 7) / 8);
  const int passes = (items + kThreads - 1) / kThreads;
  return dim3((unsigned)tokens, (unsigned)std::max(1, std::min(passes, 1024 / tokens)));
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" int alpx_rotary_append_rows(const void* query, const void* key, const void* value,
                                       void* query_out, void* key_rows, void* value_rows,
                                       int64_t pool_rows, const int32_t* slots,
                                       const int32_t* positions, int dtype, int tokens,
                                       int q_heads, int kv_heads, int head_dim, int value_dim,
                                       int rotary_dim, int style, double frequency_base,
                                       double frequency_scale, void* stream) {
  const char* what = "alpx_rotary_append_rows";
  RotaryArgs a = {};
  const int status = rotary_args(what, a, query, key, value, query_out, key_rows, value_rows,
                                 slots, positions, dtype, tokens, q_heads, kv_heads, head_dim,
                                 value_dim, rotary_dim, style, frequency_base, frequency_scale);
  if (status != ALPX_OK) return status;
  if (pool_rows <= 0) return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  a.rows = pool_rows;
  const uintptr_t align = (uintptr_t)query | (uintptr_t)key | (uintptr_t)value |
                          (uintptr_t)query_out | (uintptr_t)key_rows | (uintptr_t)value_rows;
  a.vec = head_dim % 8 == 0 && value_dim % 8 == 0 && (align & 15) == 0;
  a.pvec = a.vec && a.R % 8 == 0;
  const void* kernel = dtype == ALPX_F32   ? (const void*)rotary_rows_kernel<float>
                       : dtype == ALPX_F16 ? (const void*)rotary_rows_kernel<f16_t>
                                           : (const void*)rotary_rows_kernel<bf16_t>;
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_KV_APPEND, s);
  void* args[] = {&a};
  (void)hipLaunchKernel(kernel, rotary_grid(a, tokens), dim3(kThreads), args, 0, s);
  return check_launch(what);
}

extern "C" int alpx_q4_append_rows(const void* query, const void* key, const void* value,
                                   void* query_out, void* key_codes, void* key_scales,
                                   void* value_codes, void* value_scales, int page_size,
                                   int num_pages, const int32_t* slots, const int32_t* positions,
                                   int dtype, int tokens, int q_heads, int kv_heads, int head_dim,
                                   int rotary_dim, int style, double frequency_base,
                                   double frequency_scale, void* stream) {
  const char* what = "alpx_q4_append_rows";
  RotaryArgs a = {};
  const int status = rotary_args(what, a, query, key, value, query_out, key_codes, value_codes,
                                 slots, positions, dtype, tokens, q_heads, kv_heads, head_dim,
                                 head_dim, rotary_dim, style, frequency_base, frequency_scale);
  if (status != ALPX_OK) return status;
  if (!key_scales || !value_scales) return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!q4_dim_ok(head_dim)) return fail(ALPX_EUNSUPPORTED, "%s: head width must be 64, 96, 128 or 256", what);
  if (num_pages <= 0) return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (!power_of_two(page_size) || page_size < 32)
    return fail(ALPX_EINVAL, "page_size must be a power of two of at least 32");
  if ((int64_t)num_pages * page_size > 0x7fffffff)
    return fail(ALPX_EUNSUPPORTED, "%s: 2^31 rows or more", what);
  if ((((uintptr_t)key_codes | (uintptr_t)value_codes | (uintptr_t)key_scales |
        (uintptr_t)value_scales) & 15) != 0)
    return fail(ALPX_EINVAL, "%s: codes and scales must be 16-byte aligned", what);
  a.ks = (f16_t*)key_scales;
  a.vs = (f16_t*)value_scales;
  a.rows = (int64_t)num_pages * page_size;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  const uintptr_t align = (uintptr_t)query | (uintptr_t)key | (uintptr_t)value | (uintptr_t)query_out;
  a.vec = (align & 15) == 0;
  a.pvec = a.vec && a.R % 8 == 0;
  const void* kernel = dtype == ALPX_F32   ? (const void*)q4_append_kernel<float>
                       : dtype == ALPX_F16 ? (const void*)q4_append_kernel<f16_t>
                                           : (const void*)q4_append_kernel<bf16_t>;
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_KV_APPEND, s);
  void* args[] = {&a};
  (void)hipLaunchKernel(kernel, rotary_grid(a, tokens), dim3(kThreads), args, 0, s);
  return check_launch(what);
}

extern "C" int alpx_q4_rows(const void* key_codes, const void* key_scales, const void* value_codes,
                            const void* value_scales, int page_size, int num_pages,
                            const int32_t* slots, int rows, int kv_heads, int head_dim,
                            void* key_out, void* value_out, int out_dtype, void* stream) {
  const char* what = "alpx_q4_rows";
  if (!key_codes || !key_scales || !value_codes || !value_scales || !slots || !key_out || !value_out)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(out_dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (rows <= 0 || kv_heads <= 0 || num_pages <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (!q4_dim_ok(head_dim)) return fail(ALPX_EUNSUPPORTED, "%s: head width must be 64, 96, 128 or 256", what);
  if (!power_of_two(page_size) || page_size < 32)
    return fail(ALPX_EINVAL, "page_size must be a power of two of at least 32");
  if ((int64_t)num_pages * page_size > 0x7fffffff)
    return fail(ALPX_EUNSUPPORTED, "%s: 2^31 rows or more", what);
  if ((((uintptr_t)key_codes | (uintptr_t)value_codes | (uintptr_t)key_scales |
        (uintptr_t)value_scales | (uintptr_t)key_out | (uintptr_t)value_out) & 15) != 0)
    return fail(ALPX_EINVAL, "%s: codes, scales and rows must be 16-byte aligned", what);
  Q4RowsArgs a = {};
  a.codes[0] = (const uint32_t*)key_codes;
  a.codes[1] = (const uint32_t*)value_codes;
  a.scales[0] = (const f16_t*)key_scales;
  a.scales[1] = (const f16_t*)value_scales;
  a.out[0] = key_out;
  a.out[1] = value_out;
  a.slots = slots;
  a.rows = (int64_t)num_pages * page_size;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.items = (int64_t)rows * kv_heads * (head_dim / 8);
  const int span = kThreads * (out_dtype == ALPX_F32 ? kFlight<float> : kFlight<bf16_t>);
  const unsigned blocks = (unsigned)std::min<int64_t>((a.items + span - 1) / span, 1 << 20);
  const void* kernel = out_dtype == ALPX_F32   ? (const void*)q4_rows_kernel<float>
                       : out_dtype == ALPX_F16 ? (const void*)q4_rows_kernel<f16_t>
                                               : (const void*)q4_rows_kernel<bf16_t>;
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_AUX, s);
  void* args[] = {&a};
  (void)hipLaunchKernel(kernel, dim3(blocks, 2), dim3(kThreads), args, 0, s);
  return check_launch(what);
}
