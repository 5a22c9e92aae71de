// A page pool of 4-bit codes.
//
// The pool of K (and one like it of V) is two arrays:
//   codes  [num_pages, kv_heads, page_size, D / 2] bytes: channel c of a row
//          is the low (c even) or high half of byte c / 2;
//   scales [num_pages, kv_heads, 2, D / 32, page_size] float16: the steps,
//          then the least values, of 32 channels each.
// Channel c of a row stands for least + step * code.  A page keeps a head's
// rows side by side, so an attention block, which reads one head, reads whole
// lines; steps lie along the rows, the order in which the products of the
// attention want them.  5 bits a value in all.
#pragma once

#include "alpx_common.h"

namespace alpx {

constexpr int kQ4Group = 32;  // channels that share a step and a least value
constexpr int kQ4Rows = 32;   // rows of an attention tile, all of one page
constexpr int kQ4Waves = 4;   // of an attention block; they take its steps in turn

inline bool q4_dim_ok(int d) { return d == 64 || d == 96 || d == 128 || d == 256; }
// Whether n bytes at a and m bytes at b (null: none) meet.
inline bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  return a && b && (uintptr_t)a < (uintptr_t)b + (uintptr_t)m &&
         (uintptr_t)b < (uintptr_t)a + (uintptr_t)n;
}

inline bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

// The attention's arguments, which its kernels share whatever the type of q.
struct Q4Args {
  const void* q;     // [B, N, Hq, D]
  const char* kc;    // codes and scales of the pool
  const char* ks;
  const char* vc;
  const char* vs;
  const int32_t* table;   // [B, max_pages]
  const int32_t* prefix;  // [B]
  const int32_t* counts;  // [B] or null
  const void* gate;       // null, or [B, N, Hq, D]
  void* out;              // [B, N, Hq, D]
  int page_shift, max_pages, num_pages;
  int length, batch, nodes, q_heads, kv_heads, group;
  int col_tiles;      // column tiles per (sequence, kv head)
  int slots;          // shares of the rows per (kv head, column tile)
  float* part_o;      // segments of O, [segment, kv head, column][D]
  float2* part_st;    // reference score and sum of P of their columns
  int4* found;        // [batch]: first and last slot of a sequence, P, end; null:
                      // a slot takes a whole sequence, and there is no join
  float scale_log2;
  int out_dtype;
  int vec;            // q, gate and out may be read and written in vectors
};

struct Q4Kernel {
  const void* fn;
  const void* join;
  int join_cols;
  int cols;    // columns per block
  int rows;    // rows per step
  int per_cu;  // blocks on a CU at a time
};

// The kernel for queries of one type (q4_f32.hip, q4_f16.hip, q4_bf16.hip:
// apart, so that they compile side by side).
Q4Kernel q4_kernel_f32(int head_dim, int cols);
Q4Kernel q4_kernel_f16(int head_dim, int cols);
Q4Kernel q4_kernel_bf16(int head_dim, int cols);

}  // namespace alpx
