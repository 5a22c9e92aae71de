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

inline bool q4_dim_ok(int d) { return d == 64 || d == 96 || d == 128 || d == 256; }
// Whether n bytes at a and m bytes at b (null: none) meet.
inline bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  return a && b && (uintptr_t)a < (uintptr_t)b + (uintptr_t)m &&
         (uintptr_t)b < (uintptr_t)a + (uintptr_t)n;
}

inline bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace alpx
