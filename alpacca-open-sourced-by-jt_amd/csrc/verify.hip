// Which drafted tokens stand, from given random numbers.
//
// Draft 0 of a sequence is the token that it holds already; draft i, a child
// of draft parents[i], was proposed as the token behind it.  p = target[i] is
// the target's distribution behind draft i, q = draft[i] the distribution
// that the children of i were drawn from, one after the other and each from
// all of q.  From draft 0 on, the children x_1, x_2, ... of a draft are tried
// in rising order, with r_0 = p, Z_0 = 1:
//   child j stands if u_j q(x_j) Z < r(x_j); the walk goes on from it;
//   else r <- max(r - Z q, 0), Z <- sum r, and the next child is tried;
// and where no child stands (or none is left), the last token is drawn from
// r: the first x whose running sum exceeds u_0 sum r.  Tokens then follow the
// target's distribution exactly.  Children that no distribution drew (draft
// null) stand with probability r(x) / Z, which takes x out of p when refused:
//   child j stands if u_j Z < r(x_j); else r(x_j) <- 0, Z <- Z - r(x_j).
// If nothing is left of r, p itself is drawn from; if p holds nothing either,
// the last token is -1.  Entries that are not positive and finite weigh 0.
//
// Sums run in float64: a running sum in float32 would be off by more than a
// small token's weight.
//
// Bound by the one or two rows of the vocabulary that the last token is drawn
// from.  One launch gathers the drafts' own entries, walks as far as it can
// without a sum (in every block for itself: a walk is short) and leaves the
// sums of slices of the row, a wave a slice; a second finds the slice and the
// token.  64 x 6 drafts over 131101 tokens, float32: 67 MB in 25.8 us, 18 of them
// the sums (3.7 TB/s: every block first walks, two chains of dependent reads of
// some 3 us), 8 the draw, which no read of a row bounds.
#include <math.h>

#include <algorithm>

#include "alpx_common.h"
#include "timing.h"

namespace alpx {
namespace {

constexpr int kMostDrafts = 1024;
constexpr int kMostSlices = 256;  // four per lane
constexpr int kSumThreads = 256, kDrawThreads = 512;
constexpr int kRounds = 4;       // launches of sums, for trees of drawn drafts

struct Stand {  // where a walk stopped
  int last;      // the draft that it reached
  int from;      // the next child to try, from here on
  int tried;     // children of `last` refused so far
  int accepted;  // drafts that stand; 0: the sequence has no drafts
  int more;      // a sum is wanted, and then there is another child to try
};

struct VerifyArgs {
  const int32_t* tokens;   // [B, N]
  const void* target;      // [B, N, V]
  const void* draft;       // [B, N, V] or null
  const int32_t* parents;  // [B, N] or null (chains)
  const int32_t* counts;   // [B] or null
  const float* uniforms;   // [B, N]
  int32_t* paths;          // [B, N]
  int32_t* accepted;       // [B]
  int32_t* out;            // [B, N]
  double* sums;            // [2][B, slices]: of this round and the one before
  Stand* stands;           // [2][B]
  double* zs;              // [B, N]: Z of the refusals where a walk stopped
  int64_t vocab, slice;    // tokens; tokens of a slice
  int nodes, slices, batch;
  int round;               // of a launch; of the draw: the last one
};

__device__ __forceinline__ float weight(float x) {
  return x > 0.f && x < __builtin_inff() ? x : 0.f;
}

// What a block knows of a sequence's drafts, in LDS as large as they are.
struct Drafts {
  double* z;   // [N] Z of the refusals at the draft that the walk is at
  float* p;    // [N] the parent's distributions at the token
  float* q;
  float* u;
  int* up;     // [N] parent, -1: never reached
  int* token;
  int* gone;   // [N] tokens refused there (draft null)
  struct Shared {
    Stand at;
    int ngone;
  };
  Shared* s;
};

__host__ __device__ inline size_t drafts_bytes(int nodes) {
  return (size_t)nodes * 32 + sizeof(Drafts::Shared);
}

__device__ __forceinline__ Drafts drafts_in(char* lds, int nodes) {
  Drafts d;
  d.z = (double*)lds;
  d.p = (float*)(d.z + nodes);
  d.q = d.p + nodes;
  d.u = d.q + nodes;
  d.up = (int*)(d.u + nodes);
  d.token = d.up + nodes;
  d.gone = d.token + nodes;
  d.s = (Drafts::Shared*)(d.gone + nodes);
  return d;
}

template <typename T>
__device__ __forceinline__ void gather(const VerifyArgs& a, int b, int count, const Drafts& d) {
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const int64_t at = (int64_t)b * a.nodes + i;
    int up = a.parents != nullptr ? a.parents[at] : i - 1;
    if (up < 0 || up >= i) up = -1;
    const int x = a.tokens[at];
    float p = 0.f, q = 1.f;
    if (up >= 0) {
      const int64_t row = ((int64_t)b * a.nodes + up) * a.vocab;
      const bool in = x >= 0 && x < a.vocab;
      p = in ? weight(to_f32(((const T*)a.target)[row + x])) : 0.f;
      if (a.draft != nullptr) q = in ? weight(to_f32(((const T*)a.draft)[row + x])) : 0.f;
    }
    d.up[i] = up;
    d.token[i] = x;
    d.p[i] = p;
    d.q[i] = q;
    d.u[i] = a.uniforms[at];
  }
}

// What `tried` refusals leave of p where the draft has q.
__device__ __forceinline__ double left_of(double p, double q, const double* z, int tried) {
  double r = p;
  for (int j = 0; j < tried; ++j) r = fmax(r - z[j] * q, 0.0);
  return r;
}

// Goes on from d.s->at until a draft refuses a child or none is left.  One
// wave; z[0 .. tried] are the sums known so far (z[0] = 1).  The drafts that
// stand enter the sequence's path.
template <bool DRAFT>
__device__ __forceinline__ void walk(const VerifyArgs& a, int b, int count, const Drafts& d) {
  const int lane = threadIdx.x & 63;
  int last = d.s->at.last, from = d.s->at.from, tried = d.s->at.tried, accepted = d.s->at.accepted;
  double rem = 1.0;  // draft null: 1 less the tokens refused here
  bool refused = false, more = false;
  while (true) {
    int child = -1;
    for (int i0 = from & ~63; i0 < count && child < 0; i0 += 64) {
      const int i = i0 + lane;
      const unsigned long long hit = __ballot(i >= from && i < count && d.up[i] == last);
      if (hit != 0) child = i0 + __ffsll((long long)hit) - 1;
    }
    if (DRAFT && refused) {
      more = child >= 0;
      break;
    }
    if (child < 0) break;
    const int x = d.token[child];
    const double u = (double)d.u[child];
    double w;
    bool stands;
    if constexpr (DRAFT) {
      const double q = (double)d.q[child];
      w = left_of((double)d.p[child], q, d.z, tried);
      stands = u * q * d.z[tried] < w;
    } else {
      bool again = false;  // a token that was refused here once weighs nothing
      for (int j0 = 0; j0 < tried; j0 += 64)
        again |= __ballot(j0 + lane < tried && d.gone[j0 + lane] == x) != 0;
      w = again ? 0.0 : (double)d.p[child];
      stands = u * rem < w;
    }
    from = child + 1;
    if (stands) {
      if (lane == 0 && a.paths != nullptr) {
        a.paths[(int64_t)b * a.nodes + accepted] = child;
        a.out[(int64_t)b * a.nodes + accepted - 1] = x;
      }
      ++accepted;
      last = child;
      tried = 0;
      rem = 1.0;
      continue;
    }
    rem -= w;
    if (lane == 0) d.gone[tried] = x;
    __builtin_amdgcn_wave_barrier();  // (LDS traffic of a wave runs in order)
    ++tried;
    refused = true;
  }
  if (lane == 0) d.s->at = Stand{last, from, tried, accepted, more};
}

// A thread's share of the weights x0 <= x < x1 of a row: p where nothing was
// refused, else what the refusals left.  d.gone[0 .. ngone) are the tokens of
// the range that weigh nothing.
template <typename T, bool DRAFT>
__device__ __forceinline__ double range_sum(const T* p, const T* q, int64_t x0, int64_t x1,
                                            const Drafts& d, int tried, int ngone, int thread,
                                            int threads) {
  constexpr int VN = 16 / (int)sizeof(T);
  struct alignas(16) Unit {
    T x[VN];
  };
  double sum = 0.0;
  auto one = [&](int64_t x) __attribute__((always_inline)) {
    float w = weight(to_f32(p[x]));
    if constexpr (DRAFT) {
      sum += tried == 0 ? (double)w
                        : left_of((double)w, (double)weight(to_f32(q[x])), d.z, tried);
    } else {
      for (int j = 0; j < ngone; ++j)
        if (d.gone[j] == x) w = 0.f;
      sum += (double)w;
    }
  };
  int64_t v0 = x0, v1 = x0;  // whole units
  if (!DRAFT || (((uintptr_t)p ^ (uintptr_t)q) & 15) == 0) {
    const int64_t head = (int64_t)((0u - (unsigned)((uintptr_t)(p + x0) & 15)) & 15) / (int)sizeof(T);
    v0 = x0 + head < x1 ? x0 + head : x1;
    v1 = v0 + (x1 - v0) / VN * VN;
  }
  for (int64_t x = x0 + thread; x < v0; x += threads) one(x);
  constexpr int kFlight = 4;  // units on their way
  for (int64_t first = v0 + (int64_t)thread * VN; first < v1; first += (int64_t)threads * VN * kFlight) {
    Unit pu[kFlight], qu[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int64_t x = min(first + (int64_t)i * threads * VN, v1 - VN);  // past the last: again, unused
      pu[i] = *(const Unit*)(p + x);
      if (DRAFT && tried != 0) qu[i] = *(const Unit*)(q + x);
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int64_t x = first + (int64_t)i * threads * VN;
      if (x >= v1) break;
      float w[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) w[e] = weight(to_f32(pu[i].x[e]));
      if constexpr (DRAFT) {
        if (tried != 0) {
#pragma unroll
          for (int e = 0; e < VN; ++e)
            sum += left_of((double)w[e], (double)weight(to_f32(qu[i].x[e])), d.z, tried);
          continue;
        }
      } else {
        for (int j = 0; j < ngone; ++j) {
#pragma unroll
          for (int e = 0; e < VN; ++e)
            if (d.gone[j] == x + e) w[e] = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < VN; ++e) sum += (double)w[e];
    }
  }
  for (int64_t x = v1 + thread; x < x1; x += threads) one(x);
  return sum;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

// The refused tokens of draft d.s->at.last that lie in [x0, x1), in d.gone: all
// of its children, since none stands.
__device__ __forceinline__ void gone_in(int count, int64_t x0, int64_t x1, const Drafts& d) {
  if (threadIdx.x == 0) d.s->ngone = 0;
  __syncthreads();
  const int last = d.s->at.last;
  for (int i = threadIdx.x; i < count; i += blockDim.x)
    if (d.up[i] == last && d.token[i] >= x0 && d.token[i] < x1)
      d.gone[atomicAdd(&d.s->ngone, 1)] = d.token[i];
  __syncthreads();
}

__device__ __forceinline__ int count_of(const VerifyArgs& a, int b) {
  return a.counts != nullptr ? min(max(a.counts[b], 0), a.nodes) : a.nodes;
}

__device__ __forceinline__ void slice_of(const VerifyArgs& a, int s, int64_t& x0, int64_t& x1) {
  x0 = min(s * a.slice, a.vocab);
  x1 = min(x0 + a.slice, a.vocab);
}

// Running sums of the slices: a lane has those of its four, of which `s` are
// the sums; every wave for itself.  Returns the sum of all.
__device__ __forceinline__ double slice_scan(const double* sums, int slices, int lane, double (&s)[4],
                                             double (&upto)[4]) {
  double run = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = 4 * lane + i < slices ? sums[4 * lane + i] : 0.0;
    run += s[i];
  }
  double x = run;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o = __shfl_up(x, off);
    if (lane >= off) x += o;
  }
  double before = __shfl_up(x, 1);
  if (lane == 0) before = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before += s[i];
    upto[i] = before;
  }
  return __shfl(upto[3], 63);
}

// Grid (slices / waves, B).  Round 0 walks from draft 0; the next ones, for
// trees of drawn drafts, go on from where a sum was wanted: another refusal's
// sum by the whole device, where the draw's block alone would form it (trees of
// 8 x 12 drafts over 131101 tokens, float32: 137 us with 1 round, 78 with 2,
// 31 with 4, 36 with 6, and 1.2 us a round that no sequence needs).  Refusals of
// one draft's children past the fourth are that block's alone, and each forms
// all before it again: 11, 23 and 63 refused in a row over 131101 tokens, float32,
// take 1.1, 4.4 and 30 ms.
template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kSumThreads) verify_sums(VerifyArgs a) {
  constexpr int kWaves = kSumThreads / 64;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Drafts d = drafts_in(lds, a.nodes);
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool writes = blockIdx.x == 0;
  const int count = count_of(a, b);
  const int64_t row0 = (int64_t)b * a.nodes;
  const int now = DRAFT ? a.round & 1 : 0;
  Stand* const stand = a.stands + (int64_t)now * a.batch + b;
  double* const sums = a.sums + ((int64_t)now * a.batch + b) * a.slices;
  const int s = blockIdx.x * kWaves + wave;
  Stand start = {0, 1, 0, count > 0 ? 1 : 0, count > 0};
  if (!DRAFT || a.round == 0) {
    if (writes) {
      for (int i = tid; i < a.nodes; i += kSumThreads) {
        a.paths[row0 + i] = i == 0 && count > 0 ? 0 : -1;
        a.out[row0 + i] = -1;
      }
    }
  } else {
    start = a.stands[(int64_t)(now ^ 1) * a.batch + b];
  }
  const double* const old = a.sums + ((int64_t)(now ^ 1) * a.batch + b) * a.slices;
  if (!start.more) {  // it has what it needs
    if (writes && tid == 0) *stand = start;
    if (DRAFT && a.round > 0 && s < a.slices && lane == 0) sums[s] = old[s];
    return;
  }
  gather<T>(a, b, count, d);
  if (DRAFT && a.round > 0) {
    for (int i = tid; i < start.tried; i += kSumThreads) d.z[i] = a.zs[row0 + i];
    if (wave == 0) {
      double own[4], upto[4];
      const double z = slice_scan(old, a.slices, lane, own, upto);
      if (lane == 0) {
        d.z[start.tried] = z;
        if (writes) a.zs[row0 + start.tried] = z;
      }
    }
  } else if (DRAFT && tid == 0) {
    d.z[0] = 1.0;
    if (writes) a.zs[row0] = 1.0;
  }
  if (tid == 0) d.s->at = start;
  __syncthreads();
  if (wave == 0) {
    VerifyArgs mine = a;
    if (!writes) mine.paths = nullptr;
    walk<DRAFT>(mine, b, count, d);
  }
  __syncthreads();
  const Stand at = d.s->at;
  if (writes && tid == 0) *stand = at;
  int64_t x0, x1;
  slice_of(a, s, x0, x1);
  if (!DRAFT) {  // of all the block's slices
    int64_t y0, y1, y2, y3;
    slice_of(a, blockIdx.x * kWaves, y0, y1);
    slice_of(a, blockIdx.x * kWaves + kWaves - 1, y2, y3);
    gone_in(count, y0, y3, d);
  }
  if (s >= a.slices) return;
  const int64_t row = (row0 + at.last) * a.vocab;
  const double sum = wave_sum(range_sum<T, DRAFT>((const T*)a.target + row, (const T*)a.draft + row,
                                                  x0, x1, d, at.tried, DRAFT ? 0 : d.s->ngone, lane, 64));
  if (lane == 0) sums[s] = sum;
}

// Grid (B).
template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kDrawThreads) verify_draw(VerifyArgs a) {
  constexpr int kWaves = kDrawThreads / 64;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Drafts d = drafts_in(lds, a.nodes);
  __shared__ double sums[kMostSlices], part[kWaves];
  __shared__ int64_t found[2][kWaves];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = count_of(a, b);
  const int64_t row0 = (int64_t)b * a.nodes;
  const int now = DRAFT ? a.round & 1 : 0;
  const Stand first = a.stands[(int64_t)now * a.batch + b];
  const float u0 = a.uniforms[row0];
  if (tid < a.slices) sums[tid] = a.sums[((int64_t)now * a.batch + b) * a.slices + tid];
  if (first.accepted == 0) {
    if (tid == 0) a.accepted[b] = 0;
    return;
  }
  if (tid == 0) d.s->at = first;
  if (DRAFT)
    for (int i = tid; i < max(first.tried, 1); i += kDrawThreads) d.z[i] = a.zs[row0 + i];
  if (!DRAFT) {  // the refused tokens
    for (int i = tid; i < count; i += kDrawThreads) {
      int up = a.parents != nullptr ? a.parents[row0 + i] : i - 1;
      if (up < 0 || up >= i) up = -1;
      d.up[i] = up;
      d.token[i] = a.tokens[row0 + i];
    }
  }
  __syncthreads();
  double own[4], upto[4];  // of this lane's slices
  // the sums of all slices by this block alone, a wave a slice
  auto sum_all = [&](int tried, int ngone) __attribute__((always_inline)) {
    __syncthreads();
    const int64_t row = (row0 + d.s->at.last) * a.vocab;
    for (int s = wave; s < a.slices; s += kWaves) {
      int64_t x0, x1;
      slice_of(a, s, x0, x1);
      const double sum = wave_sum(range_sum<T, DRAFT>((const T*)a.target + row,
                                                      (const T*)a.draft + row, x0, x1, d, tried,
                                                      ngone, lane, 64));
      if (lane == 0) sums[s] = sum;
    }
    __syncthreads();
  };
  if constexpr (DRAFT) {
    bool gathered = false;
    // the sum of what the last refusal left is there: try the next child
    while (d.s->at.more) {
      if (!gathered) gather<T>(a, b, count, d);
      gathered = true;
      const double z = slice_scan(sums, a.slices, lane, own, upto);
      const Stand before = d.s->at;
      __syncthreads();
      if (tid == 0) d.z[before.tried] = z;
      __syncthreads();
      if (wave == 0) walk<DRAFT>(a, b, count, d);
      __syncthreads();
      sum_all(d.s->at.tried, 0);
    }
    __syncthreads();
  }
  const Stand at = d.s->at;
  int tried = at.tried;
  double z = slice_scan(sums, a.slices, lane, own, upto);
  bool plain = false;  // draw from p itself
  if (!(z > 0.0) && tried > 0) {
    plain = true;
    tried = 0;
    sum_all(0, 0);
    z = slice_scan(sums, a.slices, lane, own, upto);
  }
  int64_t token = -1;
  if (z > 0.0) {
    const double t = fmax((double)u0 * z, 0.0);
    // the slice: the first whose running sum exceeds t, or the last that has any
    int mine = -1, last = -1;
    double before = 0.0, at_last = 0.0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      if (!(own[i] > 0.0)) continue;
      if (last < 0) {
        last = 4 * lane + i;
        at_last = upto[i] - own[i];
      }
      if (upto[i] > t) {
        mine = 4 * lane + i;
        before = upto[i] - own[i];
      }
    }
    const unsigned long long over = __ballot(mine >= 0), some_at = __ballot(last >= 0);
    const bool inside = over != 0;
    const int from = inside ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some_at);
    const int slice = __shfl(inside ? mine : last, from);
    before = __shfl(inside ? before : at_last, from);
    int64_t x0, x1;
    slice_of(a, slice, x0, x1);
    if (!DRAFT && !plain) gone_in(count, x0, x1, d);
    const int ngone = DRAFT || plain ? 0 : d.s->ngone;
    const int64_t row = (row0 + at.last) * a.vocab;
    const T* p = (const T*)a.target + row;
    const T* q = (const T*)a.draft + row;
    auto left = [&](int64_t x) __attribute__((always_inline)) {
      float w = weight(to_f32(p[x]));
      if constexpr (DRAFT) {
        if (tried > 0) return left_of((double)w, (double)weight(to_f32(q[x])), d.z, tried);
      } else {
        for (int j = 0; j < ngone; ++j)
          if (d.gone[j] == x) w = 0.f;
      }
      return (double)w;
    };
    // neighbouring tokens to a thread, threads in order; the first kKept are
    // asked for together (whose sum passes t goes over all of its own again)
    constexpr int kKept = 4;
    const int64_t per = (x1 - x0 + kDrawThreads - 1) / kDrawThreads;
    const int64_t m0 = min(x0 + tid * per, x1), m1 = min(m0 + per, x1);
    double kept[kKept], sum = 0.0;
    int64_t some = -1;
#pragma unroll
    for (int i = 0; i < kKept; ++i) kept[i] = m0 + i < m1 ? left(m0 + i) : 0.0;
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      sum += kept[i];
      if (kept[i] > 0.0) some = m0 + i;
    }
    for (int64_t x = m0 + kKept; x < m1; ++x) {
      const double w = left(x);
      sum += w;
      if (w > 0.0) some = x;
    }
    double run = sum;  // inclusive, in the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double o = __shfl_up(run, off);
      if (lane >= off) run += o;
    }
    if (lane == 63) part[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += part[w];
    int64_t hit = INT64_MAX;
    if (inside && before + run > t) {
      double c = before + (run - sum);
      for (int64_t x = m0; x < m1; ++x) {
        const double w = left(x);
        c += w;
        if (w > 0.0 && c > t) {
          hit = x;
          break;
        }
      }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const int64_t h = __shfl_xor(hit, off), l = __shfl_xor(some, off);
      hit = h < hit ? h : hit;
      some = l > some ? l : some;
    }
    if (lane == 0) {
      found[0][wave] = hit;
      found[1][wave] = some;
    }
    __syncthreads();
    // (rounding alone, or u of 1 and more, leave t behind the last weight)
    for (int w = 0; w < kWaves; ++w) {
      hit = found[0][w] < hit ? found[0][w] : hit;
      some = found[1][w] > some ? found[1][w] : some;
    }
    token = hit != INT64_MAX ? hit : some;
  }
  if (tid == 0) {
    a.accepted[b] = at.accepted;
    a.out[row0 + at.accepted - 1] = (int32_t)token;
  }
}

// About 4096 slices in all, a wave each, of 256 tokens at least (131101 tokens,
// 64 x 6 float32 and 32 x 24 bf16: 26.6 and 15.1 us with 8192 slices, 25.8 and
// 13.3 with 4096, 29.7 and 14.6 with 2048; 1 x 8 over 32768: 10.1 us with slices
// of 128 and 256, 10.7 with 512, 11.6 with 1024).
void slicing(int batch, int64_t vocab, int64_t& slice, int& slices) {
  const int64_t want = std::max(4, std::min(kMostSlices, 4096 / batch));
  slice = std::max<int64_t>(256, ((vocab + want - 1) / want + 63) / 64 * 64);
  slices = (int)((vocab + slice - 1) / slice);
}

bool sizes_ok(int batch, int nodes, int64_t vocab) {
  return batch > 0 && batch <= 65535 && nodes > 0 && nodes <= kMostDrafts && vocab > 0 &&
         vocab <= 0x7fffffff;
}

template <typename T>
void launch(VerifyArgs a, int batch, int rounds, hipStream_t s) {
  const dim3 grid((unsigned)((a.slices + kSumThreads / 64 - 1) / (kSumThreads / 64)), (unsigned)batch);
  const size_t lds = drafts_bytes(a.nodes);
  if (a.draft != nullptr) {
    for (a.round = 0; a.round < rounds; ++a.round)
      hipLaunchKernelGGL((verify_sums<T, true>), grid, dim3(kSumThreads), lds, s, a);
    a.round = rounds - 1;
    hipLaunchKernelGGL((verify_draw<T, true>), dim3((unsigned)batch), dim3(kDrawThreads), lds, s, a);
  } else {
    hipLaunchKernelGGL((verify_sums<T, false>), grid, dim3(kSumThreads), lds, s, a);
    hipLaunchKernelGGL((verify_draw<T, false>), dim3((unsigned)batch), dim3(kDrawThreads), lds, s, a);
  }
}

}  // namespace
}  // namespace alpx

using namespace alpx;

extern "C" size_t alpx_verify_workspace_bytes(int batch, int nodes, int64_t vocab) {
  if (!sizes_ok(batch, nodes, vocab)) return 0;
  int64_t slice;
  int slices;
  slicing(batch, vocab, slice, slices);
  return (size_t)batch * (2 * (sizeof(Stand) + (size_t)slices * sizeof(double)) +
                          (size_t)nodes * sizeof(double));
}

extern "C" int alpx_verify_drafts(const int32_t* tokens, const void* target, const void* draft,
                                  const int32_t* parents, const int32_t* counts,
                                  const float* uniforms, int32_t* paths, int32_t* accepted,
                                  int32_t* new_tokens, void* workspace, size_t workspace_bytes,
                                  int batch, int nodes, int64_t vocab, int dtype, void* stream) {
  const char* what = "alpx_verify_drafts";
  if (!tokens || !target || !uniforms || !paths || !accepted || !new_tokens)
    return fail(ALPX_EINVAL, "%s: null buffer", what);
  if (!dtype_ok(dtype)) return fail(ALPX_EINVAL, "%s: unknown dtype", what);
  if (batch <= 0 || nodes <= 0 || vocab <= 0)
    return fail(ALPX_EINVAL, "%s: sizes must be positive", what);
  if (!sizes_ok(batch, nodes, vocab))
    return fail(ALPX_EUNSUPPORTED, "%s: at most 65535 sequences, %d drafts and 2^31 - 1 tokens",
                what, kMostDrafts);
  const size_t need = alpx_verify_workspace_bytes(batch, nodes, vocab);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)
    return fail(ALPX_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace", what, need);
  VerifyArgs a = {};
  a.tokens = tokens;
  a.target = target;
  a.draft = draft;
  a.parents = parents;
  a.counts = counts;
  a.uniforms = uniforms;
  a.paths = paths;
  a.accepted = accepted;
  a.out = new_tokens;
  a.stands = (Stand*)workspace;
  a.zs = (double*)(a.stands + 2 * (size_t)batch);
  a.sums = a.zs + (size_t)batch * nodes;
  a.vocab = vocab;
  a.nodes = nodes;
  a.batch = batch;
  slicing(batch, vocab, a.slice, a.slices);
  // a chain's first refusal is its last
  const int rounds = draft && parents ? std::min(nodes, kRounds) : 1;
  hipStream_t s = (hipStream_t)stream;
  TimedRegion timed(ALPX_T_AUX, s);
  switch (dtype) {
    case ALPX_F32: launch<float>(a, batch, rounds, s); break;
    case ALPX_F16: launch<f16_t>(a, batch, rounds, s); break;
    default: launch<bf16_t>(a, batch, rounds, s); break;
  }
  return check_launch(what);
}
