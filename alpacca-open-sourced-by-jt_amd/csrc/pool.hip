// Page pool bookkeeping and the rows of drafted tokens, on the device: block
// tables, free pages and slots from request lengths (paged_resize), the
// visibility masks of draft trees (tree_masks), and the accepted path's rows
// moved up behind the prefix (tree_commit).
#include <algorithm>

#include "alpx_common.h"
#include "timing.h"
#include "wave_scan.h"

namespace alpx {
namespace {

// A uniform load through the scalar cache (no block of the launch writes
// what it reads).
__device__ __forceinline__ int load_const(const int32_t* p) {
  return __builtin_amdgcn_readfirstlane(
      *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p);
}

// ------------------------------------------------------------------ resize

// Up to this many rows one launch does it all: the block's own loop over the
// rows costs less than a second launch.
constexpr int kOneLaunchRows = 4096;

struct ResizeArgs {
  int32_t* table;    // [B, max_pages]
  int32_t* lengths;  // [B]
  int32_t* free;     // [num_pages], a stack
  int32_t* count;    // [1], pages on the stack
  const int32_t* targets;  // [B]
  int32_t* starts;   // [B + 1]
  int32_t* slots;    // [tokens]
  int32_t* positions;
  int32_t* sequences;
  int32_t* granted;  // [B]
  int32_t* scratch;  // [B + 1]: pages taken by the sequences before; the stack's height
  int batch, max_pages, page_shift, num_pages, tokens;
  bool expand;       // this launch writes the rows' slots too
};

constexpr int kThreads = 1024;  // largest block
constexpr int kFlight = 4;      // pages a thread moves at a time

// Inclusive sums over a block of NT threads, of one value per thread, and
// the sum of all.  A wave's sums meet the others' in `part` (two of them in
// turn, so that one barrier a call is enough).
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t (*part)[kThreads / 64], int& turn,
                                              int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_inclusive(x);
  int64_t* p = part[turn];
  turn ^= 1;
  if (lane == 63) p[wave] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll 4
  for (int w = 0; w < NT / 64; ++w) {
    const int64_t s = p[w];
    if (w < wave) before += s;
    all += s;
  }
  total = all;
  return x + before;
}

// What sequence b asks for.
struct Change {
  bool valid;
  int length, target;  // target = length where the request is refused
  int old_pages, new_pages;
};

__device__ __forceinline__ Change change_of(const ResizeArgs& a, int b) {
  Change c = {};
  if (b >= a.batch) return c;
  const int64_t cap = (int64_t)a.max_pages << a.page_shift;
  const int len = a.lengths[b], target = a.targets[b];
  c.valid = len >= 0 && len <= cap && target >= 0 && target <= cap;
  c.length = len;
  c.target = c.valid ? target : len;
  const int round = (1 << a.page_shift) - 1;
  c.old_pages = c.valid ? (int)(((int64_t)len + round) >> a.page_shift) : 0;
  c.new_pages = c.valid ? (int)(((int64_t)target + round) >> a.page_shift) : 0;
  return c;
}

// Largest i < n with start[i] <= x (start[0] <= x).
__device__ __forceinline__ int find_last(const int32_t* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Slot, position and sequence of new row t.  A page that the sequence held
// comes from its table, a new one off the stack; the row that begins a new
// page enters it in the table.
__device__ __forceinline__ void write_row(const ResizeArgs& a, const int32_t* start, int t,
                                          int total, int64_t have) {
  int slot = -1, pos = -1, b = -1;
  if (t < total) {
    b = find_last(start, a.batch, t);
    const int held = a.lengths[b] - (start[b + 1] - start[b]);  // rows before this call
    pos = held + t - start[b];
    const int round = (1 << a.page_shift) - 1;
    const int held_pages = (int)(((int64_t)held + round) >> a.page_shift);
    const int c = pos >> a.page_shift;
    int32_t* entry = a.table + (int64_t)b * a.max_pages + c;
    int page;
    if (c < held_pages) {
      page = *entry;
    } else {
      const int64_t place = have - 1 - ((int64_t)a.scratch[b] + c - held_pages);
      page = place >= 0 && place < a.num_pages ? a.free[place] : -1;
      if ((pos & round) == 0) *entry = page;
    }
    slot = (page << a.page_shift) + (pos & round);
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
  a.sequences[t] = b;
}

// One block: sums over the sequences give every page that is released its
// place on the stack and every page that is taken its place below the top.
// Released page r of R (in the order of sequences, then rows) goes to place
// count + R - 1 - r, and taken page t comes from place count + R - 1 - t, so
// that cutting sequences back by what they just grew restores the stack.
// A request that needs pages is granted while the sum of the pages needed up
// to it is at most what the stack holds (and its new rows end within
// `tokens`): a refused one makes later ones that need pages be refused too.
// Released pages move in flat order over the block, whatever each sequence's
// share; taken ones with the rows that begin them.
//
// A tile is NT sequences; more of them go tile by tile.  Sums of pages fit 32
// bits per tile (max_pages <= 2^20) and share a 64-bit sum; sums of rows run
// over refused requests, which need not fit, in 64 bits.  Bound by latency:
// a handful of dependent round trips to memory and block-wide sums.
template <int NT>
__global__ void __launch_bounds__(NT) resize_kernel(ResizeArgs a) {
  __shared__ int64_t part[2][kThreads / 64];
  __shared__ int32_t first[NT], table_at[NT];
  __shared__ int32_t starts[NT + 1];
  const int tid = threadIdx.x;
  const int tiles = (a.batch + NT - 1) / NT;
  const int64_t count = max(*a.count, 0);
  int turn = 0;
  int64_t total;

  // released pages (low half) and needed ones (high half) of the tile
  const Change c0 = change_of(a, tid);
  auto pages_of = [](const Change& c) {
    const int64_t need = max(c.new_pages - c.old_pages, 0);
    return need << 32 | (uint32_t)max(c.old_pages - c.new_pages, 0);
  };
  const int64_t incl0 = block_scan<NT>(pages_of(c0), part, turn, total);
  const int64_t total0 = total;
  int64_t R = (uint32_t)total0;
  for (int t = 1; t < tiles; ++t) {
    block_scan<NT>(pages_of(change_of(a, t * NT + tid)), part, turn, total);
    R += (uint32_t)total;
  }
  // the released pages onto the stack
  if (R > 0) {
    int64_t base = 0;
    for (int t = 0; t < tiles; ++t) {
      const Change c = t == 0 ? c0 : change_of(a, t * NT + tid);
      const int out = (uint32_t)pages_of(c);
      int64_t incl = incl0;
      total = total0;
      if (t > 0) incl = block_scan<NT>(pages_of(c), part, turn, total);
      first[tid] = (int)(uint32_t)incl - out;
      table_at[tid] = c.new_pages;
      __syncthreads();
      const int here = (int)(uint32_t)total;
      for (int i0 = tid; i0 < here; i0 += kFlight * NT) {
        int64_t at[kFlight];
        int32_t page[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int i = min(i0 + u * NT, here - 1);
          const int s = find_last(first, NT, i);
          at[u] = (int64_t)(t * NT + s) * a.max_pages + table_at[s] + (i - first[s]);
          if (i0 + u * NT < here) page[u] = a.table[at[u]];
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int64_t place = count + R - 1 - (base + i0 + u * NT);
          if (i0 + u * NT >= here) continue;
          if (place >= 0 && place < a.num_pages) a.free[place] = page[u];
          a.table[at[u]] = -1;
        }
      }
      base += here;
      __syncthreads();
    }
  }
  // grants, and the taken pages off the stack
  const int64_t have = count + R;
  int64_t pages = 0, rows = 0, taken = 0, packed = 0;
  for (int t = 0; t < tiles; ++t) {
    const int b = t * NT + tid;
    const Change c = t == 0 ? c0 : change_of(a, b);
    const int need = max(c.new_pages - c.old_pages, 0);
    const int64_t more = max((int64_t)c.target - c.length, (int64_t)0);
    int64_t incl = incl0;
    total = total0;
    if (t > 0) incl = block_scan<NT>(pages_of(c), part, turn, total);
    const int64_t pages_to = pages + (incl >> 32);
    pages += total >> 32;
    const int64_t rows_to = rows + block_scan<NT>(more, part, turn, total);
    rows += total;
    const bool ok = c.valid && (need == 0 || pages_to <= have) && (more == 0 || rows_to <= a.tokens);
    const int take = ok ? need : 0;
    const int add = ok ? (int)more : 0;
    const int64_t both = block_scan<NT>((int64_t)take << 32 | add, part, turn, total);
    const int taken_here = (int)(total >> 32), added_here = (int)(uint32_t)total;
    const int start = (int)packed + (int)(uint32_t)both - add;
    starts[tid] = start;
    if (b < a.batch) {
      a.starts[b] = start;
      a.scratch[b] = (int)taken + (int)(both >> 32) - take;
      a.granted[b] = ok ? 1 : 0;
      if (ok && c.target != c.length) a.lengths[b] = c.target;
    }
    packed += added_here;
    if (tid == 0) starts[min(a.batch, NT)] = (int)packed;
    taken += taken_here;
  }
  if (tid == 0) {
    a.starts[a.batch] = (int)packed;
    a.scratch[a.batch] = (int)have;
    *a.count = (int)(have - taken);
  }
  if (!a.expand) return;
  __syncthreads();  // lengths, starts and scratch of every thread
  const int32_t* start = tiles > 1 ? a.starts : starts;
  for (int t = tid; t < a.tokens; t += NT) write_row(a, start, t, (int)packed, have);
}

// The new rows' slots, one thread each, in a launch of its own.
constexpr int kStaged = 4096;  // sequences whose starts fit the block's LDS
__global__ void __launch_bounds__(256) slots_kernel(ResizeArgs a) {
  __shared__ int32_t start[kStaged + 1];
  const bool staged = a.batch <= kStaged;
  if (staged) {
    for (int i = threadIdx.x; i <= a.batch; i += 256) start[i] = a.starts[i];
    __syncthreads();
  }
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  if (staged)
    write_row(a, start, t, start[a.batch], a.scratch[a.batch]);
  else
    write_row(a, a.starts, t, a.starts[a.batch], a.scratch[a.batch]);
}

// ------------------------------------------------------------------- masks

struct MaskArgs {
  const int32_t* parents;  // [B, N]
  const int32_t* counts;   // [B] or null
  const int32_t* lengths;  // [B] or null
  uint64_t* masks;         // [B, N, words]
  int32_t* depths;         // [B, N]
  int64_t* lanes;          // [B, N, 4] or null
  int nodes, words;
};

// One block per sequence, one thread per draft.  Draft i starts with itself
// and its parent; each round it takes over what the ancestor it has reached
// sees, and that one's ancestor, so a path of d steps takes log2 d rounds.
// Bound by latency: one tree of 8 drafts 2.0 us, 256 of 255 6.2 (two LDS
// round trips and a barrier a round).
template <int W>
__global__ void __launch_bounds__(W * 64) masks_kernel(MaskArgs a) {
  constexpr int N = 64 * W;
  __shared__ uint64_t sees[N][W];
  __shared__ int32_t up[N], steps[N];
  const int b = blockIdx.x, i = threadIdx.x;
  int count = a.counts != nullptr ? load_const(a.counts + b) : a.nodes;
  count = min(max(count, 0), a.nodes);
  const bool live = i < count;
  const int64_t at = (int64_t)b * a.nodes + i;
  int anc = live ? a.parents[at] : -1;
  if (anc < 0 || anc >= i) anc = -1;
  int depth = anc >= 0 ? 1 : 0;
  uint64_t mine[W];
#pragma unroll
  for (int w = 0; w < W; ++w) mine[w] = live && (i >> 6) == w ? 1ull << (i & 63) : 0ull;
  for (int round = 0; round < 11; ++round) {  // paths of up to 2^10 steps
    if (!__syncthreads_or(anc >= 0)) break;   // and last round's reads are done
#pragma unroll
    for (int w = 0; w < W; ++w) sees[i][w] = mine[w];
    up[i] = anc;
    steps[i] = depth;
    __syncthreads();
    if (anc >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) mine[w] |= sees[anc][w];
      depth += steps[anc];
      anc = up[anc];
    }
  }
  if (i >= a.nodes) return;
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < a.words) a.masks[at * a.words + w] = mine[w];
  a.depths[at] = live ? depth : -1;
  if (a.lanes != nullptr) {
    const int64_t p = live ? (int64_t)load_const(a.lengths + b) + depth : 0;
    typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
    i64x2* dst = (i64x2*)(a.lanes + 4 * at);
    dst[0] = (i64x2){p, p};
    dst[1] = (i64x2){p, 0};
  }
}

// ------------------------------------------------------------------ commit

struct CommitArgs {
  void* k;
  void* v;
  const int32_t* pages;   // [B, max_pages], or null: contiguous caches
  const int32_t* paths;   // [B, M]
  const int32_t* accepted;  // [B]
  const int32_t* prefix;  // [B]
  int64_t ks_pos, ks_b, vs_pos, vs_b;  // bytes between rows, and pages (or sequences)
  int64_t capacity;       // rows of a sequence
  int k_units, v_units;   // copy units per row
  int max_pages, page_shift, num_pages, path_max;
};

// Address of logical row `row` of sequence b, null past the capacity and
// where the table names no page of the pool.
__device__ __forceinline__ char* commit_row(const CommitArgs& a, char* base, int b, int64_t row,
                                            int64_t pos, int64_t outer) {
  if (row >= a.capacity) return nullptr;
  if (a.pages == nullptr) return base + b * outer + row * pos;
  const int pg = a.pages[(int64_t)b * a.max_pages + (row >> a.page_shift)];
  if (pg < 0 || pg >= a.num_pages) return nullptr;
  return base + pg * outer + (row & ((1 << a.page_shift) - 1)) * pos;
}

// Row P + path[i] moves to row P + i.  A path names drafts in rising order,
// so path[i] >= i, and ends where it stops rising.  A block has all rows of
// its units, kChunk steps at a time: it reads their rows, meets, and writes.
// Step i reads a row at or past P + i, and the chunks before it wrote rows
// before that, so no row is written before it has been read.  Bound by
// latency: path, table, row, one round trip each (one thread per unit that
// took its rows in turn, eight at a time: 9.4 us for 128 sequences of up to
// 16 accepted drafts, 32 KiB each; this one 4.2).
constexpr int kUnits = 64, kSteps = 4;          // units of a block, steps of a thread
constexpr int kChunk = 256 / kUnits * kSteps;   // steps of a block at a time
static_assert(kChunk <= 64, "a wave holds a chunk's steps in its lanes");

template <typename X>
__global__ void __launch_bounds__(256) commit_kernel(CommitArgs a) {
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z == 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int unit = blockIdx.x * kUnits + lane;
  const int units = is_v ? a.v_units : a.k_units;
  const int64_t P = load_const(a.prefix + b);
  const int n = min(load_const(a.accepted + b), a.path_max);
  if (P < 0 || (int)blockIdx.x * kUnits >= units) return;  // the whole block
  char* base = (char*)(is_v ? a.v : a.k);
  const int64_t pos = is_v ? a.vs_pos : a.ks_pos, outer = is_v ? a.vs_b : a.ks_b;
  const int32_t* path = a.paths + (int64_t)b * a.path_max;
  int last = -1;
  for (int i0 = 0; i0 < n; i0 += kChunk) {
    // lane l holds step i0 + l, and where its rows lie
    const int from = i0 + lane < n && lane < kChunk ? path[i0 + lane] : -1;
    const int before = lane == 0 ? last : __shfl_up(from, 1);
    const unsigned long long fall = __ballot(from <= before || from < 0);  // bit kChunk is set
    const int steps = min(__ffsll((long long)fall) - 1, kChunk);
    last = __shfl(from, kChunk - 1);
    const bool moves = lane < steps && from != i0 + lane;
    char* src = moves ? commit_row(a, base, b, P + from, pos, outer) : nullptr;
    char* dst = moves ? commit_row(a, base, b, P + i0 + lane, pos, outer) : nullptr;
    if (src == nullptr) dst = nullptr;
    if (dst == nullptr) src = nullptr;
    X x[kSteps];
    char* to[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int l = wave * kSteps + j;  // this wave's steps
      const char* p = (const char*)__shfl((long long)src, l);
      to[j] = (char*)__shfl((long long)dst, l);
      if (unit >= units) to[j] = nullptr;
      if (to[j] != nullptr) x[j] = *(const X*)(p + (int64_t)unit * sizeof(X));
    }
    __syncthreads();  // every row of the chunk is read
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
      if (to[j] != nullptr) *(X*)(to[j] + (int64_t)unit * sizeof(X)) = x[j];
    if (steps < kChunk) return;  // the path has ended
    __syncthreads();
  }
}

int commit_launch(const char* what, CommitArgs a, int dtype, int batch, int kv_heads, int key_dim,
                  int value_dim, void* stream) {
  const int64_t es = (int64_t)dtype_size(dtype);
  const int64_t kb = kv_heads * (int64_t)key_dim * es, vb = kv_heads * (int64_t)value_dim * es;
  const uintptr_t align = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)kb | (uintptr_t)vb |
                          (uintptr_t)a.ks_pos | (uintptr_t)a.vs_pos | (uintptr_t)a.ks_b |
                          (uintptr_t)a.vs_b;
  const int64_t size = (align & 15) == 0 ? 16 : es;
  if (std::max(kb, vb) / size > 0x3fffffff) return fail(ALPX_EUNSUPPORTED, "%s: rows too long", what);
  a.k_units = (int)(kb / size);
  a.v_units = (int)(vb / size);
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_KV_APPEND, s);
  for (int b0 = 0; b0 < batch; b0 += 65535) {  // grid y
    CommitArgs c = a;
    c.paths += (int64_t)b0 * a.path_max;
    c.accepted += b0;
    c.prefix += b0;
    if (a.pages != nullptr)
      c.pages += (int64_t)b0 * a.max_pages;
    else {
      c.k = (char*)a.k + b0 * a.ks_b;
      c.v = (char*)a.v + b0 * a.vs_b;
    }
    const dim3 grid((unsigned)((std::max(a.k_units, a.v_units) + kUnits - 1) / kUnits),
                    (unsigned)std::min(batch - b0, 65535), 2);
    if (size == 16)
      hipLaunchKernelGGL(commit_kernel<u32x4>, grid, dim3(256), 0, s, c);
    else if (es == 4)
      hipLaunchKernelGGL(commit_kernel<uint32_t>, grid, dim3(256), 0, s, c);
    else
      hipLaunchKernelGGL(commit_kernel<uint16_t>, grid, dim3(256), 0, s, c);
  }
  return check_launch(what);
}

bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" int alpx_paged_resize(int32_t* block_table, int32_t* lengths, int32_t* free_pages,
                                 int32_t* free_count, const int32_t* targets, int batch,
                                 int max_pages, int page_size, int num_pages, int tokens,
                                 int32_t* starts, int32_t* slots, int32_t* positions,
                                 int32_t* sequences, int32_t* granted, int32_t* scratch,
                                 void* stream) {
  const char* what = "alpx_paged_resize";
  if (!block_table || !lengths || !free_pages || !free_count || !targets || !starts || !granted ||
      !scratch || (tokens > 0 && (!slots || !positions || !sequences)))
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (batch <= 0 || max_pages <= 0 || num_pages <= 0 || tokens < 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (!power_of_two(page_size)) return fail(ALPX_EINVAL, "page_size must be a power of two");
  if ((int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > 0x7fffffff)
    return fail(ALPX_EUNSUPPORTED, "%s: 2^31 rows or more", what);
  if (max_pages > 1 << 20) return fail(ALPX_EUNSUPPORTED, "%s: more than 2^20 pages a sequence", what);
  // (the new rows' launch counts its threads in 31 bits)
  if (tokens > 0x7fffffff - 255) return fail(ALPX_EUNSUPPORTED, "%s: more than 2^31 - 256 tokens", what);
  ResizeArgs a = {block_table, lengths,   free_pages, free_count, targets,
                  starts,      slots,     positions,  sequences,  granted, scratch,
                  batch,       max_pages, __builtin_ctz((unsigned)page_size), num_pages, tokens,
                  tokens <= kOneLaunchRows};
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_AUX, s);
  // a block as large as the work that it finds
  if (batch <= 256 && tokens <= 1024)
    hipLaunchKernelGGL(resize_kernel<256>, dim3(1), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(resize_kernel<kThreads>, dim3(1), dim3(kThreads), 0, s, a);
  if (!a.expand)
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)((tokens + 255) / 256)), dim3(256), 0, s, a);
  return check_launch(what);
}

extern "C" int alpx_tree_masks(const int32_t* parents, const int32_t* counts,
                               const int32_t* lengths, uint64_t* masks, int32_t* depths,
                               int64_t* position_lanes, int batch, int nodes, int mask_words,
                               void* stream) {
  const char* what = "alpx_tree_masks";
  if (!parents || !masks || !depths || (position_lanes && !lengths))
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (batch <= 0 || nodes <= 0) return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (mask_words != (nodes + 63) / 64)
    return fail(ALPX_EINVAL, "%s: mask_words must be ceil(nodes / 64)", what);
  if (nodes > 1024) return fail(ALPX_EUNSUPPORTED, "%s: more than 1024 drafts", what);
  if (((uintptr_t)position_lanes & 15) != 0)
    return fail(ALPX_EINVAL, "%s: position lanes must be 16-byte aligned", what);
  const MaskArgs a = {parents, counts, lengths, masks, depths, position_lanes, nodes, mask_words};
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_AUX, s);
  const dim3 grid((unsigned)batch);
  if (mask_words <= 1)
    hipLaunchKernelGGL(masks_kernel<1>, grid, dim3(64), 0, s, a);
  else if (mask_words <= 2)
    hipLaunchKernelGGL(masks_kernel<2>, grid, dim3(128), 0, s, a);
  else if (mask_words <= 4)
    hipLaunchKernelGGL(masks_kernel<4>, grid, dim3(256), 0, s, a);
  else if (mask_words <= 8)
    hipLaunchKernelGGL(masks_kernel<8>, grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL(masks_kernel<16>, grid, dim3(1024), 0, s, a);
  return check_launch(what);
}

extern "C" int alpx_tree_commit(void* key_cache, void* value_cache, const int32_t* paths,
                                const int32_t* accepted, const int32_t* prefix_lens, int dtype,
                                int64_t capacity, int batch, int kv_heads, int key_dim,
                                int value_dim, int path_max, void* stream) {
  const char* what = "alpx_tree_commit";
  if (!key_cache || !value_cache || !paths || !accepted || !prefix_lens)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (capacity <= 0 || batch <= 0 || kv_heads <= 0 || key_dim <= 0 || value_dim <= 0 ||
      path_max <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  CommitArgs a = {};
  a.k = key_cache;
  a.v = value_cache;
  a.paths = paths;
  a.accepted = accepted;
  a.prefix = prefix_lens;
  a.path_max = path_max;
  a.capacity = capacity;
  const int64_t es = (int64_t)dtype_size(dtype);
  a.ks_b = kv_heads * (int64_t)key_dim * es;
  a.vs_b = kv_heads * (int64_t)value_dim * es;
  a.ks_pos = batch * a.ks_b;
  a.vs_pos = batch * a.vs_b;
  return commit_launch(what, a, dtype, batch, kv_heads, key_dim, value_dim, stream);
}

extern "C" int alpx_tree_commit_paged(void* key_pages, void* value_pages,
                                      const int32_t* block_table, int max_pages, int page_size,
                                      int num_pages, const int32_t* paths,
                                      const int32_t* accepted, const int32_t* prefix_lens,
                                      int dtype, int batch, int kv_heads, int key_dim,
                                      int value_dim, int path_max, void* stream) {
  const char* what = "alpx_tree_commit_paged";
  if (!key_pages || !value_pages || !block_table || !paths || !accepted || !prefix_lens)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (max_pages <= 0 || num_pages <= 0 || batch <= 0 || kv_heads <= 0 || key_dim <= 0 ||
      value_dim <= 0 || path_max <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (!power_of_two(page_size)) return fail(ALPX_EINVAL, "page_size must be a power of two");
  CommitArgs a = {};
  a.k = key_pages;
  a.v = value_pages;
  a.pages = block_table;
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.paths = paths;
  a.accepted = accepted;
  a.prefix = prefix_lens;
  a.path_max = path_max;
  a.capacity = (int64_t)max_pages * page_size;
  const int64_t es = (int64_t)dtype_size(dtype);
  a.ks_pos = kv_heads * (int64_t)key_dim * es;
  a.vs_pos = kv_heads * (int64_t)value_dim * es;
  a.ks_b = a.ks_pos * page_size;
  a.vs_b = a.vs_pos * page_size;
  return commit_launch(what, a, dtype, batch, kv_heads, key_dim, value_dim, stream);
}
