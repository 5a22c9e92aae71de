// Entry points of the attention over a page pool of 4-bit codes: which kernel,
// and over how many shares of the rows (the mathematics: q4_kernel.h).
#include <math.h>

#include <algorithm>

#include "alpx_common.h"
#include "prefill_run.h"
#include "q4_internal.h"
#include "timing.h"

namespace alpx {
namespace {

constexpr int kCus = 256;

// Up to this length of the longest sequence a block takes a whole sequence and
// one launch is all: with few blocks, and with one for every CU.  bf16, 32/8
// heads of 128, us whole and split:
//   1 x 1 token on 512 rows 8.8, 10.4; on 1024 12.8, 10.8; on 2048 20.7, 11.0
//   32 x 1      on 512 10.4, 13.2; on 2048 23.3, 25.1; on 4096 38.2, 33.0
//   4 x 64      on 512 17.4, 24.1; on 2048 41.1, 40.3; on 8192 134, 101
constexpr int64_t kAloneRows = 512, kAloneRowsFull = 2048;
// Beyond a block a CU a share has this many rows at least: 32 x 1 on 512 rows,
// split: 13.2 us with 128 and 256, 23.4 with 512; 4 x 1 on 2048: 13.0 with 128,
// 11.3 with 256 and more.
constexpr int64_t kRowsPerSlot = 256;

struct Q4Plan {
  Q4Kernel kernel;
  int col_tiles, slots;
  bool alone;
  size_t segments, bytes;  // columns' segments, bytes in all
  int64_t blocks, joins;
};

Q4Plan q4_plan(int batch, int nodes, int q_heads, int kv_heads, int head_dim, int length, int dtype) {
  Q4Plan p = {};
  const int cols = nodes * (q_heads / kv_heads);
  p.kernel = dtype == ALPX_F32   ? q4_kernel_f32(head_dim, cols)
             : dtype == ALPX_F16 ? q4_kernel_f16(head_dim, cols)
                                 : q4_kernel_bf16(head_dim, cols);
  p.col_tiles = (cols + p.kernel.cols - 1) / p.kernel.cols;
  const int64_t steps = (length + p.kernel.rows - 1) / p.kernel.rows;
  const int64_t tiles = (int64_t)batch * steps;
  const int64_t units = (int64_t)kv_heads * p.col_tiles;
  const int64_t share = std::min(kCus * p.kernel.per_cu / units,
                                 std::max(kCus / units, tiles * p.kernel.rows / kRowsPerSlot));
  p.slots = (int)std::min(std::max<int64_t>(share, 1), tiles);
  p.alone = length <= (batch * units >= kCus ? kAloneRowsFull : kAloneRows);
  if (p.alone) p.slots = batch;
  p.blocks = ((int64_t)p.slots * kv_heads + kXcds - 1) / kXcds * kXcds * p.col_tiles;
  if (p.alone) return p;
  p.segments = (size_t)(p.slots + batch) * kv_heads * p.col_tiles * p.kernel.cols;
  p.bytes = p.segments * ((size_t)head_dim * 4 + sizeof(float2)) + (size_t)batch * sizeof(int4);
  p.joins = (int64_t)batch * kv_heads * ((cols + p.kernel.join_cols - 1) / p.kernel.join_cols);
  return p;
}

// Sums of tiles, also rounded up to whole runs of every slot, and threads of
// a launch stay in 31 and 32 bits.
bool sizes_ok(int batch, int nodes, int q_heads, int kv_heads, int head_dim, int length, int dtype) {
  if (batch <= 0 || nodes <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 ||
      length <= 0 || !q4_dim_ok(head_dim) || !dtype_ok(dtype))
    return false;
  if (length > (1 << 30) || (int64_t)batch * ((int64_t)length / kQ4Rows + 1) >= ((int64_t)1 << 31) - 2048)
    return false;
  if ((int64_t)nodes * (q_heads / kv_heads) > (1 << 24) || batch > (1 << 24) || kv_heads > (1 << 20))
    return false;
  const Q4Plan p = q4_plan(batch, nodes, q_heads, kv_heads, head_dim, length, dtype);
  return p.blocks * 64 * kQ4Waves <= 0xffffffff && p.joins * 2 * head_dim <= 0xffffffff;
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" size_t alpx_q4_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                          int head_dim, int length, int dtype) {
  if (!sizes_ok(batch, nodes, q_heads, kv_heads, head_dim, length, dtype)) return 0;
  return q4_plan(batch, nodes, q_heads, kv_heads, head_dim, length, dtype).bytes;
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
  if (page_size > 1 << 24) return fail(ALPX_EUNSUPPORTED, "%s: pages of more than 2^24 rows", what);
  if (length > (int64_t)max_pages * page_size)
    return fail(ALPX_ERANGE, "%s: length exceeds the block table", what);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(ALPX_EINVAL, "scale must be positive and finite");
  if (!sizes_ok(batch, nodes, q_heads, kv_heads, head_dim, length, dtype))
    return fail(ALPX_EUNSUPPORTED, "%s: too many rows, tokens or sequences", what);
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
  const Q4Plan p = q4_plan(batch, nodes, q_heads, kv_heads, head_dim, length, dtype);
  Q4Args a = {};
  a.q = q;
  a.kc = (const char*)key_codes;
  a.ks = (const char*)key_scales;
  a.vc = (const char*)value_codes;
  a.vs = (const char*)value_scales;
  a.table = block_table;
  a.prefix = prefix_lens;
  a.counts = counts;
  a.gate = gate;
  a.out = out;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.length = length;
  a.batch = batch;
  a.nodes = nodes;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.col_tiles = p.col_tiles;
  a.slots = p.slots;
  a.scale_log2 = scale * kLog2e;
  a.out_dtype = out_dtype;
  a.vec = (((uintptr_t)q | (uintptr_t)out) & 15) == 0;
  a.part_o = (float*)workspace;
  a.part_st = (float2*)(a.part_o + p.segments * head_dim);
  a.found = p.alone ? nullptr : (int4*)(a.part_st + p.segments);
  hipStream_t s = (hipStream_t)stream;
  {
    TimedRegion timed(ALPX_T_DECODE, s);
    void* args[] = {&a};
    (void)hipLaunchKernel(p.kernel.fn, dim3((unsigned)p.blocks), dim3(64 * kQ4Waves), args, 0, s);
  }
  if (p.alone) return check_launch(what);
  TimedRegion timed(ALPX_T_DECODE_COMBINE, s);
  int cols = nodes * a.group, tile_cols = p.kernel.cols;
  void* args[] = {&a, &cols, &tile_cols};
  (void)hipLaunchKernel(p.kernel.join, dim3((unsigned)p.joins), dim3(2 * head_dim), args, 0, s);
  return check_launch(what);
}
