// Beam search's selection (gfx950; contract in batch_ops.h): of a request's beams and their logits the n continuations
// with the largest score s_i + l_iv - log sum_v exp l_iv. The reference decodes one sequence greedily
// (python/nanoserve/qwen.py:166-177) and has no counterpart.
//
// Within a beam the order is that of its logits, so the rows are read once and nothing of their length is written:
//  * rows: a workgroup takes a part of one row, keeps the part's n largest logits and its maximum and sum of
//    exponentials. The n-th largest of a tile's 256 thread maxima is reached by n logits of that tile, so only
//    those from it on can be among its n largest: hardly more than are kept. Bounds come from bit-wise ballots, not from a
//    sort, and every wave finds the workgroup's by itself from LDS: each wave's own n-th of 64 lets three times as many
//    logits through, and of n = 64 nearly all (4 beams of 152064 with n 64 302 us, 24 now; 16 x 8 beams 27.2, 25.7).
//  * merge: a workgroup per request bounds the parts' lists the same way, by entry `depth` of each, and orders what is left
//    by rank; lists of many equal sums are joined beam by beam, a list to a lane, then the beams' lists.
// Bound by HBM and by the bounds' and lists' instructions in turn: 16 x 8 beams of 151936 fp32 25.7 us, of them 19.7 the rows
// (78 MB, 4.0 TB/s) and 5 the merge's latency; 4 beams of 152064 bf16 10.7, two launches' latency. Tiles of 2 vectors
// to a thread take 37.7 for the 16 x 8, of 8 more registers than five workgroups of a CU have.
// Keys are (logit, lowest index first), so equal logits never make a list longer than its bound. Scores are compared
// in 64 bits: two beams' continuations are often closer than a step of fp32 at their size.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "batch_ops.h"
#include "logit_rows.h"
#include "spans.h"
#include "w4_kernels.h"

namespace ns {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMostVecs = 4;                     // vectors of 8 logits of a thread in a tile
constexpr int kMostBeams = 64, kMostKept = 64;   // a list to a lane
constexpr int kMostParts = 64;
// Threads (in the merge: lists) beyond n that may reach a bound. us with 2, 4 and 8: 8 x 8 beams of 151936 bf16 21.8, 17.1, 17.6.
constexpr int kSlack = 4;
constexpr int kAtOnce = 8;                       // comparisons whose operands are loaded together
static_assert(kWaves == 4, "the end of beam_rows_kernel");
constexpr int kMostKeys = 12288;                 // keys of all parts of a request in the merge's LDS

struct BeamArgs {
  const void* logits;
  long long row_stride;
  const float* scores;
  uint64_t* keys;    // [rows][parts][n]: logit key, complement of the index; 0: none
  double2* sums;     // [rows][parts]: maximum, sum of exp(l - maximum)
  float* out_scores;
  int *out_tokens, *out_parents;
  int V, beams, n, parts, tiles;  // (tiles of a row)
  int segment;                    // keys of a wave's list of a tile
};

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  auto up = [](uint32_t x, auto ctrl, auto rows) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using M = std::integral_constant<int, 0xf>;
  v = up(v, std::integral_constant<int, 0x111>{}, M{});
  v = up(v, std::integral_constant<int, 0x112>{}, M{});
  v = up(v, std::integral_constant<int, 0x114>{}, M{});
  v = up(v, std::integral_constant<int, 0x118>{}, M{});
  v = up(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  v = up(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// How many of the lanes' values, `groups` each, reach x.
template <int N>
__device__ __forceinline__ int reach_of(const uint32_t (&h)[N], int groups, uint32_t x) {
  int k = 0;
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (u < groups) k += __popcll(__ballot(h[u] >= x));
  return k;
}

// A value that n of the lanes' values reach (0: fewer than n are not 0), and how many reach it: at most `slack` more, or
// as many as are equal to the n-th. Searched from the highest bit in which they differ. most: the largest.
template <int N>
__device__ __forceinline__ uint32_t nth_value(const uint32_t (&h)[N], int groups, int n, int slack, uint32_t most, int& reach) {
  reach = reach_of(h, groups, 1);
  if (reach < n) return 0;
  uint32_t down = 0;
#pragma unroll
  for (int u = 0; u < N; ++u) down = max(down, h[u] ? ~h[u] : 0);
  const uint32_t least = ~wave_umax(down);
  if (reach <= n + slack) return least;
  int bit = most == least ? -1 : 31 - __builtin_clz(most ^ least);
  uint32_t at = bit < 0 ? most : most & ~((2u << bit) - 1u);
#pragma unroll 1
  for (; bit >= 0; --bit) {
    const uint32_t next = at | 1u << bit;
    const int k = reach_of(h, groups, next);
    if (k < n) continue;
    at = next;
    reach = k;
    if (k <= n + slack) break;
  }
  return at;
}

// Of keys that differ in the low half: one that n of the lanes' keys reach, and no more than n, where more than n reach `at`.
template <int N>
__device__ __forceinline__ uint64_t nth_key(const uint64_t (&key)[N], uint32_t at, int n) {
  uint32_t low = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint64_t next = (uint64_t)at << 32 | low | 1u << bit;
    int k = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) k += __popcll(__ballot(key[u] >= next));
    if (k >= n) low = (uint32_t)next;
  }
  return (uint64_t)at << 32 | low;
}

// The sum over the wave's lanes, in lane 63, by DPP (row shifts, then row broadcasts).
__device__ __forceinline__ double wave_total(double v) {
  auto add = [](double x, auto ctrl, auto rows) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    auto part = [](uint32_t w) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    return x + __longlong_as_double((long long)(part((uint32_t)(u >> 32)) << 32 | part((uint32_t)u)));
  };
  using M = std::integral_constant<int, 0xf>;
  v = add(v, std::integral_constant<int, 0x111>{}, M{});
  v = add(v, std::integral_constant<int, 0x112>{}, M{});
  v = add(v, std::integral_constant<int, 0x114>{}, M{});
  v = add(v, std::integral_constant<int, 0x118>{}, M{});
  v = add(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  return add(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
}

template <typename E, int kVecs>
__global__ void __launch_bounds__(kThreads, 5) beam_rows_kernel(BeamArgs a) {
  extern __shared__ uint64_t list[];  // a.segment for each wave: keys, and kAtOnce of 0
  __shared__ uint64_t kept[2][kMostKept + kAtOnce], bests[kThreads];
  __shared__ int counts[kWaves];
  __shared__ uint32_t tops[kThreads];
  __shared__ double red_s[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long r = blockIdx.y;
  const int part = blockIdx.x, n = a.n;
  uint64_t* out = a.keys + (r * a.parts + part) * n;
  const Row<E> row{static_cast<const E*>(a.logits) + r * a.row_stride, a.V};
  const int t0 = (int)((long long)a.tiles * part / a.parts), t1 = (int)((long long)a.tiles * (part + 1) / a.parts);
  typename Row<E>::Raw raw[kVecs];
  auto fetch = [&](int t) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) raw[j] = row.fetch((t * kVecs + j) * kThreads + tid);
  };
  const float score = a.scores[r];
  fetch(t0);
  if (!(score > -INFINITY)) {  // a beam that does not count
    if (tid < n) out[tid] = 0;
    if (tid == 0) a.sums[r * a.parts + part] = make_double2(-INFINITY, 0.);
    return;
  }
  float m = -INFINITY;
  double sum = 0.;  // of this lane, in units of exp(m)
  int have = 0;     // keys in kept[now], descending
  int now = 0;
  uint64_t* segment = list + wv * a.segment;
  for (int t = t0; t < t1; ++t) {
    const int v0 = t * kVecs * kThreads + tid;
    float x[kVecs][8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      // (NaN -> -inf, +inf -> the largest finite value; -0 may stay)
      row.read(raw[j], v0 + j * kThreads, x[j], [](float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX); });
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[j][e]);
    }
    if (t + 1 < t1) fetch(t + 1);
    auto key_at = [&](int j, int e) {
      return (uint64_t)key_of(x[j][e] + 0.f) << 32 | ~(uint32_t)(row.first(v0 + j * kThreads) + e);
    };
    // The bound, which every wave finds by itself from all threads' largest
    tops[tid] = top > -INFINITY ? key_of(top + 0.f) : 0;
    __syncthreads();
    uint32_t h[kWaves], most = 0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) most = max(most, h[k] = tops[k * kWave + lane]);
    most = wave_umax(most);
    uint64_t bound = have == n ? kept[now][n - 1] + 1 : 0;
    if (have < n || reach_of(h, kWaves, (uint32_t)(bound >> 32)) > n + kSlack) {
      int reach;
      const uint32_t nth = nth_value(h, kWaves, n, kSlack, most, reach);
      uint64_t by_nth = (uint64_t)nth << 32;
      if (reach > n + kSlack) {  // many equal ones: by index too, from each thread's largest at its first place
        uint64_t best = 0;
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) best = max(best, x[j][e] == top ? key_at(j, e) : 0);
        bests[tid] = top > -INFINITY ? best : 0;
        __syncthreads();  // (all waves have found the same)
        uint64_t f[kWaves];
#pragma unroll
        for (int k = 0; k < kWaves; ++k) f[k] = bests[k * kWave + lane];
        by_nth = nth_key(f, nth, n);
      }
      bound = max(bound, by_nth);
    }
    const float least = bound >> 32 ? value_of((uint32_t)(bound >> 32)) : -FLT_MAX;
    int mine = 0;  // keys of the wave's segment: counted by ballots, so that no wave waits for a counter
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (__ballot(x[j][e] >= least)) {
          const uint64_t key = key_at(j, e);
          const bool hit = (x[j][e] >= least) & (key >= bound);
          const uint64_t hits = __ballot(hit);
          if (hit) segment[mine + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0))] = key;
          mine += __popcll(hits);
        }
    if (lane < kAtOnce) segment[mine + lane] = 0;
    if (lane == 0) counts[wv] = mine;
    if (tid < kAtOnce) kept[now][have + tid] = 0;
    if (most != 0) {
      const float mt = fmaxf(m, value_of(most));
      if (mt != m) {
        // exp(m - mt) in 32 bits, the product's rounding put right (exp of a double takes 20 registers more)
        const float d = fmaxf(m - mt, -200.f), up = d * 1.44269504f, rest = fmaf(d, 1.44269504f, -up) + d * 1.92596299e-8f;
        const float f = __builtin_amdgcn_exp2f(up);
        sum = m == -INFINITY ? 0. : sum * (double)fmaf(f, rest * 0.69314718f, f);
        m = mt;
      }
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += __expf(x[j][e] - mt);
      sum += (double)s;
    }
    __syncthreads();
    int upto[kWaves + 1] = {have};
#pragma unroll
    for (int k = 0; k < kWaves; ++k) upto[k + 1] = upto[k] + counts[k];
    const int all = upto[kWaves];
    if (all > have) {
      // ranks among the new ones and those kept before (which need not reach the bound)
      for (int i = tid; i < all; i += kThreads) {
        uint64_t key = kept[now][min(i, have)];
#pragma unroll
        for (int k = 0; k < kWaves; ++k)
          if (i >= upto[k] && i < upto[k + 1]) key = list[k * a.segment + i - upto[k]];
        int rank = 0;
        auto above = [&](const uint64_t* from, int many) {
          for (int k = 0; k < many; k += kAtOnce) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) rank += from[k + u] > key;
          }
        };
        above(kept[now], have);
#pragma unroll
        for (int k = 0; k < kWaves; ++k) above(list + k * a.segment, upto[k + 1] - upto[k]);
        if (rank < n) kept[now ^ 1][rank] = key;
      }
      now ^= 1;
      have = min(all, n);
    }
    __syncthreads();
  }
  if (tid < n) out[tid] = tid < have ? kept[now][tid] : 0;
  sum = wave_total(sum);
  if (lane == 63) red_s[wv] = sum;
  __syncthreads();
  if (tid == 0) a.sums[r * a.parts + part] = make_double2(m, (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]));
}

// The lane with the largest key, the first of several; every lane's value of it. -1: all are 0.
__device__ __forceinline__ int wave_best(uint64_t key) {
  const uint32_t hi = wave_umax((uint32_t)(key >> 32));
  uint64_t among = __ballot((uint32_t)(key >> 32) == hi);
  if (among & (among - 1)) {
    const bool in = (uint32_t)(key >> 32) == hi;
    const uint32_t lo = wave_umax(in ? (uint32_t)key : 0u);
    if (hi == 0 && lo == 0) return -1;
    among = __ballot(in && (uint32_t)key == lo);
  }
  return __builtin_ctzll(among);
}

// Unsigned order = order of the values (none of them NaN), and 0 below all.
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.);
  return b ^ (0x8000000000000000ull | (uint64_t)((int64_t)b >> 63));
}

constexpr int kMergeThreads = 512;
constexpr int kGroups = kMergeThreads / kWave;
constexpr int kUnbounded = 128;  // so many keys are ordered as they are (4 x 4 beams of 4000 9.1 us, with a bound 11.6)
constexpr int kMostRanked = kMergeThreads;  // continuations that are ordered by rank, one to a thread
constexpr int kEach = kMostKeys / kMergeThreads;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamArgs a) {
  extern __shared__ uint64_t lds[];  // [beams][parts][n], then [beams][n]
  __shared__ double base[kMostBeams];
  __shared__ uint32_t heads[kMergeThreads];
  // the sum's order, and what decides between equal sums: beam (6 bits, complement), logit key (32), index (20, complement)
  __shared__ __align__(16) ulonglong2 found[kMostRanked + kAtOnce];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.n, lists = a.beams * a.parts, all = lists * n;
  const long long r0 = (long long)blockIdx.x * a.beams;
  const uint64_t* keys = a.keys + r0 * a.parts * n;
  // the beam of list i and of key i: quotients of numbers below 2^14, exact by way of fp32 (half of one is far above its
  // error), where an integer division takes ten times the instructions
  const float per_list = 1.f / a.parts, per_key = 1.f / (a.parts * n);
  auto quotient = [](int i, float per) { return (int)(((float)i + 0.5f) * per); };
  // entry `depth` of `need` lists is reached by n continuations; both so that half of the lists are enough
  const int depth = min(n, (2 * n + lists - 1) / lists), need = (n + depth - 1) / depth;
  const uint64_t* entry = keys + depth - 1;
  uint64_t first[2], key_at[kEach];  // of the lane's lists; of its share of all keys
#pragma unroll
  for (int u = 0; u < 2; ++u) first[u] = tid + u * kMergeThreads < lists ? entry[(size_t)(tid + u * kMergeThreads) * n] : 0;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (u * kMergeThreads >= all) break;
    key_at[u] = tid + u * kMergeThreads < all ? keys[tid + u * kMergeThreads] : 0;
  }
  if (tid == 0) count = 0;
  for (int b = wv; b < a.beams; b += kMergeThreads / kWave) {
    const double2 ms = lane < a.parts ? a.sums[(r0 + b) * a.parts + lane] : make_double2(-INFINITY, 0.);
    const float score = a.scores[r0 + b];
    const double m = value_of(wave_umax(key_of((float)ms.x)));
    const double s = wave_total(ms.x > -INFINITY ? ms.y * exp(ms.x - m) : 0.);
    if (lane == 63) base[b] = (double)fminf(score, FLT_MAX) - (m + log(s));
  }
  __syncthreads();
  auto total = [&](uint64_t key, int b) { return key ? order_of(base[b] + value_of((uint32_t)(key >> 32))) : 0; };

  // A bound that n continuations reach: of the lists' entries, a list to a thread (or several: their largest)
  uint64_t bound = 1;
  if (all > kUnbounded) {
    uint64_t head = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (first[u]) head = max(head, total(first[u], quotient(tid + u * kMergeThreads, per_list)));
    for (int i = tid + 2 * kMergeThreads; i < lists; i += kMergeThreads) head = max(head, total(entry[(size_t)i * n], quotient(i, per_list)));
    heads[tid] = (uint32_t)(head >> 32);
    __syncthreads();
    const int groups = (min(lists, kMergeThreads) + kWave - 1) / kWave;
    uint32_t h[kGroups], most = 0;
#pragma unroll
    for (int u = 0; u < kGroups; ++u) most = max(most, h[u] = u < groups ? heads[u * kWave + lane] : 0);
    int reach;
    // (to the last bit where lists are few: another one that reaches the bound may bring all of its entries)
    bound = max((uint64_t)nth_value(h, groups, need, depth > 1 ? -1 : kSlack, wave_umax(most), reach) << 32, bound);
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (u * kMergeThreads >= all) break;
    const uint64_t key = key_at[u];
    const int b = min(quotient(tid + u * kMergeThreads, per_key), a.beams - 1);
    const uint64_t c = key ? total(key, b) : 0;
    if (c >= bound) {
      const int at = atomicAdd(&count, 1);
      if (at < kMostRanked)
        found[at] = make_ulonglong2(c, (uint64_t)(63 - b) << 52 | (key >> 32) << 20 | (key & 0xfffffu));
    }
  }
  __syncthreads();
  const int many = count;
  const size_t o = (size_t)blockIdx.x * n;
  if (many <= kMostRanked) {
    if (tid < kAtOnce) found[many + tid] = make_ulonglong2(0, 0);
    __syncthreads();
    if (tid < many) {
      const ulonglong2 c = found[tid];
      int rank = 0;
      for (int k = 0; k < many; k += kAtOnce) {
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const ulonglong2 x = found[k + u];
          rank += (x.x > c.x) | ((x.x == c.x) & (x.y > c.y));
        }
      }
      if (rank < n) {
        const int b = 63 - (int)(c.y >> 52);
        a.out_scores[o + rank] = (float)(base[b] + value_of((uint32_t)(c.y >> 20)));
        a.out_tokens[o + rank] = 0xfffff - (int)(c.y & 0xfffffu);
        a.out_parents[o + rank] = b;
      }
    }
    for (int k = many + tid; k < n; k += kMergeThreads) {
      a.out_scores[o + k] = -INFINITY;
      a.out_tokens[o + k] = a.out_parents[o + k] = -1;
    }
    return;
  }

  // Many equal sums: the parts' lists beam by beam, each descending, a list to a lane, then the beams' lists.
  uint64_t* best = lds + all;
#pragma unroll
  for (int u = 0; u < kEach; ++u)
    if (tid + u * kMergeThreads < all) lds[tid + u * kMergeThreads] = key_at[u];
  __syncthreads();
  for (int b = wv; b < a.beams; b += kMergeThreads / kWave) {
    const uint64_t* list = lds + ((size_t)b * a.parts + min(lane, a.parts - 1)) * n;
    uint64_t head = lane < a.parts ? list[0] : 0;
    int at = 0;
    for (int k = 0; k < n; ++k) {
      const int w = wave_best(head);
      const uint64_t key = w < 0 ? 0 : (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(head >> 32), w) << 32 |
                                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, w);
      if (lane == 0) best[b * n + k] = key;
      if (lane == w) head = ++at < n ? list[at] : 0;
    }
  }
  __syncthreads();
  if (wv != 0) return;
  const int b = min(lane, a.beams - 1);
  const uint64_t* list = best + b * n;
  uint64_t key = lane < a.beams ? list[0] : 0;
  uint64_t head = total(key, b);
  int at = 0;
  for (int k = 0; k < n; ++k) {
    const int w = wave_best(head);
    if (w < 0 ? lane == 0 : lane == w) {
      a.out_scores[o + k] = w < 0 ? -INFINITY : (float)(base[b] + value_of((uint32_t)(key >> 32)));
      a.out_tokens[o + k] = w < 0 ? -1 : (int)~(uint32_t)key;
      a.out_parents[o + k] = w;
      key = ++at < n && w >= 0 ? list[at] : 0;
      head = total(key, b);
    }
  }
}

struct Plan {
  int vecs, tiles, parts;
  size_t bytes;
};

bool sizes_ok(int R, int beams, int V, int n) {
  return R > 0 && beams > 0 && beams <= kMostBeams && V > 0 && V <= (1 << 20) && n > 0 && n <= kMostKept &&
         (long long)R * beams <= 65535;
}

Plan make_plan(int R, int beams, int V, int n) {
  Plan p;
  const long long rows = (long long)R * beams;
  auto tiles = [&](int vecs) { return (V + 8 * vecs * kThreads - 1) / (8 * vecs * kThreads); };
  // Tiles of 4 vectors to a thread where they are two workgroups to a CU and more, else of 2 (us with 2 and with 4: 16 x 8 beams
  // of 151936 fp32 37.3, 25.6; 12 x 4 of 152064 bf16 16.5, 14.3; 16 x 4 of 32000, which are 256 tiles, 11.0, 12.6). For n
  // past 32 the lists of 4 would not fit beside each other.
  p.vecs = n <= kMostKept / 2 && rows * tiles(kMostVecs) >= 512 ? kMostVecs : 2;
  p.tiles = tiles(p.vecs);
  const int want = (int)std::max(1ll, 4096 / rows);
  p.parts = std::min({p.tiles, want, kMostParts, std::max(1, kMostKeys / (beams * n))});
  p.bytes = (size_t)rows * p.parts * (n * sizeof(uint64_t) + sizeof(double2));
  return p;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_beam_select_workspace(int R, int beams, int V, int n) {
  return ns::sizes_ok(R, beams, V, n) ? ns::make_plan(R, beams, V, n).bytes : 0;
}

int ns_beam_select(const void* logits, int fp32, long long row_stride, const float* scores, float* out_scores,
                   int* out_tokens, int* out_parents, void* work, size_t work_bytes, int R, int beams, int V, int n,
                   void* stream) {
  if (!ns::sizes_ok(R, beams, V, n) || row_stride < V || row_stride >> 46) return -2;
  if (!logits || !scores || !out_scores || !out_tokens || !out_parents || !work) return -2;
  if (!ns::aligned(logits, fp32 ? 4 : 2) || !ns::aligned(work, 16)) return -2;
  for (const void* p : {(const void*)scores, (const void*)out_scores, (const void*)out_tokens, (const void*)out_parents})
    if (!ns::aligned(p, 4)) return -2;
  const ns::Plan p = ns::make_plan(R, beams, V, n);
  if (work_bytes < p.bytes) return -2;
  const size_t rows = (size_t)R * beams;
  const ns::Bytes x = ns::rows_of(logits, rows, row_stride, V, fp32 ? 4 : 2), s = ns::bytes_of(scores, 4 * rows);
  const ns::Bytes w[] = {ns::bytes_of(out_scores, 4 * (size_t)R * n), ns::bytes_of(out_tokens, 4 * (size_t)R * n),
                         ns::bytes_of(out_parents, 4 * (size_t)R * n), ns::bytes_of(work, p.bytes)};
  for (int i = 0; i < 4; ++i) {
    if (!ns::apart(w[i], x) || !ns::apart(w[i], s)) return -2;
    for (int j = 0; j < i; ++j)
      if (!ns::apart(w[i], w[j])) return -2;
  }
  ns::BeamArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.sums = reinterpret_cast<double2*>(work);
  a.keys = reinterpret_cast<uint64_t*>(a.sums + rows * p.parts);
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_parents = out_parents;
  a.V = V;
  a.beams = beams;
  a.n = n;
  a.parts = p.parts;
  a.tiles = p.tiles;
  const auto st = static_cast<hipStream_t>(stream);
  // as many threads as may reach a bound, with all of their logits
  a.segment = std::min(n + ns::kSlack, ns::kWave) * 8 * p.vecs + ns::kAtOnce;
  const size_t list = (size_t)ns::kWaves * a.segment * sizeof(uint64_t);  // (up to 37 KB)
  const dim3 grid(p.parts, (unsigned)rows);
  const auto rows_kernel = fp32 ? (p.vecs == 2 ? ns::beam_rows_kernel<float, 2> : ns::beam_rows_kernel<float, ns::kMostVecs>)
                                : (p.vecs == 2 ? ns::beam_rows_kernel<uint16_t, 2>
                                               : ns::beam_rows_kernel<uint16_t, ns::kMostVecs>);
  hipLaunchKernelGGL(rows_kernel, grid, dim3(ns::kThreads), list, st, a);
  // (its most, up to 128 KB, is asked for where 64 are not enough)
  const size_t merge = ((size_t)beams * p.parts * n + (size_t)beams * n) * sizeof(uint64_t);
  if (merge > 60 * 1024) {
    const hipError_t e = ns::cached_max_dynamic_lds(reinterpret_cast<const void*>(ns::beam_merge_kernel), 136 * 1024);
    if (e != hipSuccess) return static_cast<int>(e);
  }
  hipLaunchKernelGGL(ns::beam_merge_kernel, dim3(R), dim3(ns::kMergeThreads), merge, st, a);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
