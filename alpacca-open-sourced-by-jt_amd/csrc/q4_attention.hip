// Attention over a page pool of 4-bit codes, for one token of a sequence or a
// run of them.
//
// Sequence b holds prefix_lens[b] rows and behind them one row for each of
// its counts[b] tokens; token i sees the rows up to and with its own:
//   out[b, i, h] = softmax_j(scale * q[b, i, h] . K[j, h / G]) . V[j, h / G],
//   j <= prefix + i, K and V = least + step * code,
// times sigmoid(gate) where given.  Tokens at or past counts[b], and those
// whose row lies past `length`, give zeros.
#include <math.h>

#include <algorithm>

#include "alpx_common.h"
#include "q4_internal.h"
#include "timing.h"

namespace alpx {
namespace {

struct Q4Args {
  const void* q;     // [B, N, Hq, D]
  const uint32_t* kc;
  const f16_t* ks;
  const uint32_t* vc;
  const f16_t* vs;
  const int32_t* table;   // [B, max_pages]
  const int32_t* prefix;  // [B]
  const int32_t* counts;  // [B] or null
  const void* gate;       // null, or [B, N, Hq, D]
  void* out;              // [B, N, Hq, D]
  int page_shift, max_pages, num_pages;
  int length, nodes, q_heads, kv_heads, group, D;
  float scale_log2;
  int out_dtype;
};

constexpr int kThreads = 256, kTile = 256;

// One query head of one token per block: a tile of rows, one per thread, for
// the scores; then a channel per thread for the weighted sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) q4_simple_kernel(Q4Args a) {
  __shared__ float q[256], p[kTile], red[4];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int kvh = h / a.group, per = a.D / 8, groups = a.D / kQ4Group, size = 1 << a.page_shift;
  const int P = min(max(a.prefix[b], 0), a.length);
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.nodes) : a.nodes;
  const int end = i < count && P + i < a.length ? P + i + 1 : 0;
  const int64_t at = (((int64_t)b * a.nodes + i) * a.q_heads + h) * a.D;
  if (tid < a.D) q[tid] = to_f32(((const T*)a.q)[at + tid]) * a.scale_log2;
  __syncthreads();
  auto place = [&](int j, int64_t& head, int& row) {
    int page = a.table[(int64_t)b * a.max_pages + (j >> a.page_shift)];
    page = min(max(page, 0), a.num_pages - 1);
    head = (int64_t)page * a.kv_heads + kvh;
    row = j & (size - 1);
  };
  float top = -__builtin_inff(), sum = 0.f, o = 0.f;
  for (int j0 = 0; j0 < end; j0 += kTile) {
    float s = -__builtin_inff();
    if (j0 + tid < end) {
      int64_t head;
      int row;
      place(j0 + tid, head, row);
      s = 0.f;
      for (int w = 0; w < per; ++w) {
        const uint32_t c = a.kc[(head * size + row) * per + w];
        const f16_t* sc = a.ks + (head * 2 * groups + w / 4) * size + row;
        const float step = (float)sc[0], least = (float)sc[(int64_t)groups * size];
        for (int e = 0; e < 8; ++e)
          s = fmaf(q[8 * w + e], fmaf((float)((c >> (4 * e)) & 15u), step, least), s);
      }
    }
    float m = s;
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), top);
    const float base = m == -__builtin_inff() ? 0.f : m;
    const float alpha = top == -__builtin_inff() ? 0.f : fast_exp2(top - base);
    const float e = j0 + tid < end ? fast_exp2(s - base) : 0.f;
    p[tid] = e;
    float t = e;
    for (int off = 32; off >= 1; off >>= 1) t += __shfl_xor(t, off);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = t;
    __syncthreads();
    sum = sum * alpha + (red[0] + red[1] + red[2] + red[3]);
    top = m;
    if (tid < a.D) {
      o *= alpha;
      for (int j = 0; j < min(kTile, end - j0); ++j) {
        int64_t head;
        int row;
        place(j0 + j, head, row);
        const uint32_t c = a.vc[(head * size + row) * per + tid / 8] >> (4 * (tid & 7));
        const f16_t* sc = a.vs + (head * 2 * groups + tid / kQ4Group) * size + row;
        const float v = fmaf((float)(c & 15u), (float)sc[0], (float)sc[(int64_t)groups * size]);
        o = fmaf(p[j], v, o);
      }
    }
    __syncthreads();
  }
  if (tid < a.D) {
    float y = 0.f;
    if (end > 0) {
      y = o / sum;
      if (a.gate != nullptr) y *= fast_sigmoid(to_f32(((const T*)a.gate)[at + tid]));
    }
    if (a.out_dtype == ALPX_F32) ((float*)a.out)[at + tid] = y;
    else if (a.out_dtype == ALPX_F16) ((f16_t*)a.out)[at + tid] = from_f32<f16_t>(y);
    else ((bf16_t*)a.out)[at + tid] = from_f32<bf16_t>(y);
  }
}

bool sizes_ok(int batch, int nodes, int q_heads, int kv_heads, int head_dim, int length, int dtype) {
  return batch > 0 && nodes > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
         length > 0 && q4_dim_ok(head_dim) && dtype_ok(dtype) && batch <= 65535 && nodes <= 65535;
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" size_t alpx_q4_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                          int head_dim, int length, int dtype) {
  if (!sizes_ok(batch, nodes, q_heads, kv_heads, head_dim, length, dtype)) return 0;
  return 0;
}

extern "C" int alpx_q4_attention(const void* q, const void* key_codes, const void* key_scales,
                                 const void* value_codes, const void* value_scales,
                                 const int32_t* block_table, int max_pages, int page_size,
                                 int num_pages, const int32_t* prefix_lens, const int32_t* counts,
                                 int length, const void* gate, void* out, void* workspace,
                                 size_t workspace_bytes, int batch, int nodes, int q_heads,
                                 int kv_heads, int head_dim, float scale, int dtype, int out_dtype,
                                 void* stream) {
  const char* what = "alpx_q4_attention";
  if (!q || !key_codes || !key_scales || !value_codes || !value_scales || !block_table ||
      !prefix_lens || !out)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype) || !dtype_ok(out_dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (batch <= 0 || nodes <= 0 || q_heads <= 0 || kv_heads <= 0 || max_pages <= 0 || num_pages <= 0 ||
      length <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (q_heads % kv_heads != 0)
    return fail(ALPX_EINVAL, "attention query heads must be a multiple of KV heads");
  if (!q4_dim_ok(head_dim)) return fail(ALPX_EUNSUPPORTED, "%s: head width must be 64, 96, 128 or 256", what);
  if (!power_of_two(page_size) || page_size < 32)
    return fail(ALPX_EINVAL, "page_size must be a power of two of at least 32");
  if ((int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > 0x7fffffff)
    return fail(ALPX_EUNSUPPORTED, "%s: 2^31 rows or more", what);
  if (length > (int64_t)max_pages * page_size)
    return fail(ALPX_ERANGE, "%s: length exceeds the block table", what);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(ALPX_EINVAL, "scale must be positive and finite");
  if (!sizes_ok(batch, nodes, q_heads, kv_heads, head_dim, length, dtype))
    return fail(ALPX_EUNSUPPORTED, "%s: at most 65535 sequences and tokens of one", what);
  if ((((uintptr_t)key_codes | (uintptr_t)value_codes | (uintptr_t)key_scales |
        (uintptr_t)value_scales) & 15) != 0)
    return fail(ALPX_EINVAL, "%s: codes and scales must be 16-byte aligned", what);
  const int64_t cells = (int64_t)batch * nodes * q_heads * head_dim;
  const int64_t out_bytes = cells * (int64_t)dtype_size(out_dtype);
  const int64_t in_bytes = cells * (int64_t)dtype_size(dtype);
  if (meet(out, out_bytes, q, in_bytes) || meet(out, out_bytes, gate, in_bytes))
    return fail(ALPX_EINVAL, "%s: out must not overlap q or gate", what);
  const size_t need = alpx_q4_workspace_bytes(batch, nodes, q_heads, kv_heads, head_dim, length, dtype);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
    return fail(ALPX_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace", what, need);
  Q4Args a = {};
  a.q = q;
  a.kc = (const uint32_t*)key_codes;
  a.ks = (const f16_t*)key_scales;
  a.vc = (const uint32_t*)value_codes;
  a.vs = (const f16_t*)value_scales;
  a.table = block_table;
  a.prefix = prefix_lens;
  a.counts = counts;
  a.gate = gate;
  a.out = out;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.length = length;
  a.nodes = nodes;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.D = head_dim;
  a.scale_log2 = scale * kLog2e;
  a.out_dtype = out_dtype;
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_DECODE, s);
  const dim3 grid((unsigned)q_heads, (unsigned)nodes, (unsigned)batch);
  switch (dtype) {
    case ALPX_F32: hipLaunchKernelGGL(q4_simple_kernel<float>, grid, dim3(kThreads), 0, s, a); break;
    case ALPX_F16: hipLaunchKernelGGL(q4_simple_kernel<f16_t>, grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(q4_simple_kernel<bf16_t>, grid, dim3(kThreads), 0, s, a);
  }
  return check_launch(what);
}
