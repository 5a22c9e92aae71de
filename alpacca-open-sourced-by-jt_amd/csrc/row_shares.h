// What the kernels share that stream a cache's rows for a few tokens of each
// sequence (draft trees, 4-bit pools): whose rows a block takes, and their
// way into LDS.  The arguments A name prefix, counts, nodes, length, batch,
// slots and found as TreeArgs does.
#pragma once

#include <algorithm>

#include "alpx_common.h"
#include "prefill_run.h"
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

// Loads that may come through the scalar cache: what they read is written
// by no block of the launch.
__device__ __forceinline__ int load_const(const int32_t* p) {
  return __builtin_amdgcn_readfirstlane(
      *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p);
}

// Rows of sequence b: its prefix [0, P), its drafts [P, end).  A sequence
// without drafts has none: nobody reads its prefix.
template <typename A>
__device__ __forceinline__ void rows_from(const A& a, int prefix, int count, int& P,
                                          int& end) {
  P = min(max(prefix, 0), a.length);
  end = min(P + min(max(count, 0), a.nodes), a.length);
  if (end == P) P = end = 0;
}
template <typename A>
__device__ __forceinline__ void lane_rows(const A& a, int b, int& P, int& end) {
  rows_from(a, a.prefix[b], a.counts != nullptr ? a.counts[b] : a.nodes, P, end);
}

// The same of one sequence for the whole wave, through the scalar cache.
template <typename A>
__device__ __forceinline__ void uniform_rows(const A& a, int b, int& P, int& end) {
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
// its output and leaves no partial state (trees: a mark whether that output is
// finite).
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
template <int BK, typename A>
__device__ __forceinline__ Share find_share(const A& a, int slot, bool first_of_all) {
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

}  // namespace
}  // namespace alpx
