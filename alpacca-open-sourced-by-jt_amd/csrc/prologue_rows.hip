// The attention prologue for packed tokens of any sequences and positions:
// draft trees, whose siblings share a position, and image or video tokens,
// which have a time, a height and a width.  Every token brings its position
// lanes and the pool row that its key and value go to.
#include <algorithm>

#include "alpx_common.h"
#include "rope_internal.h"
#include "timing.h"

namespace alpx {
namespace {

struct RowsProArgs {
  const void* qg;   // [T, Hq, 2 D]: per head D query then D gate values
  const void* k;    // [T, Hkv, D]
  const void* v;    // [T, Hkv, Dv]
  const float* qw;  // [D]
  const float* kw;  // [D]
  void* q_out;      // [T, Hq, D]
  void* g_out;      // [T, Hq, D]
  void* kc;         // [rows, Hkv, D]
  void* vc;         // [rows, Hkv, Dv]
  const int32_t* slots;  // [T], rows of the pool; others write no row
  const int64_t* lanes;  // [T, 4]
  int64_t rows;
  int Hq, Hkv, D, Dv, R;
  int sec[4];
  float eps;
  double inv[kMaxPairs];
};

constexpr int kThreads = 256;

// (cos, sin) of the token's rotary pairs, formed once for all of its heads:
// an angle takes a double-precision reduction, more than the rest of a row.
__device__ __forceinline__ void token_angles(const RowsProArgs& a, int t, float2* cs) {
  for (int p = threadIdx.x; p < a.R; p += kThreads) {
    float c, s;
    rope_cs((double)a.lanes[4 * (int64_t)t + imrope_lane(p, a.sec, a.R)], a.inv[p], c, s);
    cs[p] = make_float2(c, s);
  }
}

template <typename T>
struct Row8 {
  T x[8];
};
template <typename T>
__device__ __forceinline__ Row8<T> load8(const T* p) {
  Row8<T> r;
  constexpr int kVecs = sizeof(T) * 8 / 16;
  u32x4 w[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) w[i] = ((const u32x4*)p)[i];
  __builtin_memcpy(&r, w, sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Row8<T>& r) {
  constexpr int kVecs = sizeof(T) * 8 / 16;
  u32x4 w[kVecs];
  __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < kVecs; ++i) ((u32x4*)p)[i] = w[i];
}

// One token per block row, D / 8 lanes per head row, eight channels per
// lane; grid y shares out a token's rows (query heads, key heads, value
// heads, in this order).  Dv = D, R a multiple of 8: the partner of a
// rotated channel lies R / 8 lanes away.  Bound by memory: 4133 tokens of
// 16/2 heads of 256 in bf16, 152 MB, 25.8 us = 5.9 TB/s (a copy of 1 GiB ran
// at 5.2; part of these outputs stays in cache).  8 tokens of 32/8 heads of
// 64, float32: 4.5 us, the latency of the angles and of one row.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) prologue_rows_kernel(RowsProArgs a) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  __shared__ float2 cs[D / 2];
  const int t = blockIdx.x, lane = threadIdx.x % kLanes, c0 = 8 * lane;
  const int heads = a.Hq + 2 * a.Hkv;
  const int step = kRows * gridDim.y;
  token_angles(a, t, cs);
  float qw[8], kw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qw[i] = a.qw[c0 + i];
    kw[i] = a.kw[c0 + i];
  }
  const int slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.rows;
  const int away = a.R / 8;
  const bool first = c0 < a.R, turned = c0 < 2 * a.R;
  const int partner = !turned ? 0 : (first ? away : -away);
  __syncthreads();
  for (int j0 = blockIdx.y * kRows; j0 < heads; j0 += step) {
    const int j = j0 + threadIdx.x / kLanes;
    const bool live = j < heads;
    const bool is_q = j < a.Hq, is_k = !is_q && j < a.Hq + a.Hkv;
    const int h = is_q ? j : (is_k ? j - a.Hq : j - a.Hq - a.Hkv);
    const T* src = is_q ? (const T*)a.qg + ((int64_t)t * a.Hq + h) * 2 * D
                        : (const T*)(is_k ? a.k : a.v) + ((int64_t)t * a.Hkv + h) * D;
    Row8<T> raw = {}, gate = {};
    if (live) raw = load8(src + c0);
    if (live && is_q) gate = load8(src + D + c0);
    float x[8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = to_f32(raw.x[i]);
      ss = fmaf(x[i], x[i], ss);
    }
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off);
    const float rinv = 1.f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * rinv * (is_q ? qw[i] : kw[i]);
    Row8<T> y;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float xp = __shfl(x[i], (int)(threadIdx.x & 63) + partner);
      const float2 r = cs[turned ? c0 + i - (first ? 0 : a.R) : 0];
      y.x[i] = from_f32<T>(turned ? rope_pair(first, x[i], xp, r.x, r.y) : x[i]);
    }
    if (!live) continue;
    if (is_q) {
      const int64_t at = ((int64_t)t * a.Hq + h) * D + c0;
      store8((T*)a.q_out + at, y);
      store8((T*)a.g_out + at, gate);
    } else if (stored) {
      T* dst = (T*)(is_k ? a.kc : a.vc) + ((int64_t)slot * a.Hkv + h) * D + c0;
      store8(dst, is_k ? y : raw);
    }
  }
}

// Any head widths and sections: one wave per head row, channels 64 apart,
// which loads 2 or 4 bytes a lane (4133 tokens of 16/2 heads, bf16: 256 wide
// with 33 rotary pairs 62.5 us = 2.4 TB/s against 26.7 above, 320 wide 74.8;
// 8 tokens of 32/8 heads of 80, float32: 4.5).
template <typename T>
__global__ void __launch_bounds__(kThreads) prologue_rows_any(RowsProArgs a) {
  __shared__ float2 cs[kMaxPairs];
  __shared__ float stage[kThreads / 64][kRopeMaxDim];
  const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int heads = a.Hq + 2 * a.Hkv;
  token_angles(a, t, cs);
  const int slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.rows;
  float* st = stage[wave];
  __syncthreads();
  for (int j = blockIdx.y * 4 + wave; j < heads; j += 4 * gridDim.y) {
    if (j >= a.Hq + a.Hkv) {
      const int h = j - a.Hq - a.Hkv;
      const T* src = (const T*)a.v + ((int64_t)t * a.Hkv + h) * a.Dv;
      T* dst = (T*)a.vc + ((int64_t)slot * a.Hkv + h) * a.Dv;
      if (stored)
        for (int i = lane; i < a.Dv; i += 64) dst[i] = src[i];
      continue;
    }
    const bool is_q = j < a.Hq;
    const int h = is_q ? j : j - a.Hq;
    const T* src = is_q ? (const T*)a.qg + ((int64_t)t * a.Hq + h) * 2 * a.D
                        : (const T*)a.k + ((int64_t)t * a.Hkv + h) * a.D;
    const float* w = is_q ? a.qw : a.kw;
    float ss = 0.f;
    for (int i = lane; i < a.D; i += 64) {
      const float x = to_f32(src[i]);
      ss = fmaf(x, x, ss);
    }
    ss = rope_wave_sum(ss);
    const float rinv = 1.f / sqrtf(ss / (float)a.D + a.eps);
    // LDS traffic of one wave runs in issue order: the partner reads below
    // see these stores, and the next row's stores follow them
    for (int i = lane; i < a.D; i += 64) st[i] = to_f32(src[i]) * rinv * w[i];
    __builtin_amdgcn_wave_barrier();
    const int64_t row = is_q ? (int64_t)t * a.Hq + h : (int64_t)slot * a.Hkv + h;
    T* dst = (T*)(is_q ? a.q_out : a.kc) + row * a.D;
    for (int i = lane; i < a.D; i += 64) {
      float y = st[i];
      if (i < 2 * a.R) {
        const bool first = i < a.R;
        const float2 r = cs[first ? i : i - a.R];
        y = rope_pair(first, y, st[first ? i + a.R : i - a.R], r.x, r.y);
      }
      if (is_q || stored) dst[i] = from_f32<T>(y);
      if (is_q) ((T*)a.g_out)[row * a.D + i] = src[a.D + i];
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T>
const void* pick(int D, bool fast) {
  if (!fast) return (const void*)prologue_rows_any<T>;
  return D == 64    ? (const void*)prologue_rows_kernel<T, 64>
         : D == 128 ? (const void*)prologue_rows_kernel<T, 128>
                    : (const void*)prologue_rows_kernel<T, 256>;
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" int alpx_attention_prologue_rows(const void* query_gate, const void* key,
                                            const void* value, const float* q_norm,
                                            const float* k_norm, void* query_out, void* gate_out,
                                            void* key_rows, void* value_rows, int64_t pool_rows,
                                            const int32_t* slots, const int64_t* position_lanes,
                                            int dtype, int tokens, int q_heads, int kv_heads,
                                            int head_dim, int value_dim, const int* sections,
                                            double frequency_base, float eps, void* stream) {
  const char* what = "alpx_attention_prologue_rows";
  if (!query_gate || !key || !value || !q_norm || !k_norm || !query_out || !gate_out ||
      !key_rows || !value_rows || !slots || !position_lanes || !sections)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || value_dim <= 0 ||
      pool_rows <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (q_heads % kv_heads != 0)
    return fail(ALPX_EINVAL, "attention query heads must be a multiple of KV heads");
  if (head_dim > kRopeMaxDim || value_dim > kRopeMaxDim)
    return fail(ALPX_EUNSUPPORTED, "%s: head dims above %d", what, kRopeMaxDim);
  RowsProArgs a = {};
  if (bad_sections(sections, a.R)) return fail(ALPX_EINVAL, "IMRoPE requires at least one rotary pair");
  if (head_dim < 2 * a.R)
    return fail(ALPX_EINVAL, "IMRoPE input is shorter than twice the section sum");
  if (!(frequency_base > 0.0) || !isfinite(frequency_base))
    return fail(ALPX_EINVAL, "frequency_base must be positive and finite");
  if (!(eps > 0.f) || !isfinite(eps)) return fail(ALPX_EINVAL, "epsilon must be positive and finite");
  a.qg = query_gate;
  a.k = key;
  a.v = value;
  a.qw = q_norm;
  a.kw = k_norm;
  a.q_out = query_out;
  a.g_out = gate_out;
  a.kc = key_rows;
  a.vc = value_rows;
  a.slots = slots;
  a.lanes = position_lanes;
  a.rows = pool_rows;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.Dv = value_dim;
  for (int i = 0; i < 4; ++i) a.sec[i] = sections[i];
  a.eps = eps;
  inverse_frequencies(a.inv, a.R, frequency_base, 1.0);
  const uintptr_t align = (uintptr_t)query_gate | (uintptr_t)key | (uintptr_t)value |
                          (uintptr_t)query_out | (uintptr_t)gate_out | (uintptr_t)key_rows |
                          (uintptr_t)value_rows;
  const bool fast = value_dim == head_dim && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
                    a.R % 8 == 0 && (align & 15) == 0;
  const void* kernel = dtype == ALPX_F32   ? pick<float>(head_dim, fast)
                       : dtype == ALPX_F16 ? pick<f16_t>(head_dim, fast)
                                           : pick<bf16_t>(head_dim, fast);
  // few tokens: a token's rows are shared out over blocks
  const int per = fast ? kThreads * 8 / head_dim : 4;
  const int passes = (q_heads + 2 * kv_heads + per - 1) / per;
  const int share = std::max(1, std::min(passes, 1024 / tokens));
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_LAYER, s);
  void* args[] = {&a};
  (void)hipLaunchKernel(kernel, dim3((unsigned)tokens, (unsigned)share), dim3(kThreads), args, 0, s);
  return check_launch(what);
}
