// Beam search's selection (gfx950; contract in batch_ops.h): of a request's beams and their logits the n continuations
// with the largest score s_i + l_iv - log sum_v exp l_iv. The reference decodes one sequence greedily
// (python/nanoserve/qwen.py:166-177) and has no counterpart.
//
// Within a beam the order is that of its logits, so the rows are read once and nothing of their length is written:
//  * rows: a workgroup takes a part of one row, keeps the part's n largest logits and its maximum and sum of
//    exponentials. The n-th largest of a wave's 64 lane maxima is reached by n logits of that wave, so only
//    those from the workgroup's best such bound on can be among its n largest: about as many as are kept. Bounds come
//    from bit-wise ballots, not from a sort.
//  * merge: a workgroup per request joins the parts' lists beam by beam, a list to a lane, then the beams' lists.
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
constexpr int kVecs = 2, kPer = 8 * kVecs;       // vectors and logits of a thread in a tile
constexpr int kTile = kThreads * kPer;           // logits of a tile
constexpr int kMostBeams = 64, kMostKept = 64;   // a list to a lane, and a bound from 64 lane maxima
constexpr int kMostParts = 64;
constexpr int kMostKeys = 12288;                 // keys of all parts of a request in the merge's LDS

struct BeamArgs {
  const void* logits;
  long long row_stride;
  const float* scores;
  uint64_t* keys;    // [rows][parts][n]: logit key, complement of the index; 0: none
  double2* sums;     // [rows][parts]: maximum, sum of exp(l - maximum)
  float* out_scores;
  int *out_tokens, *out_parents;
  int V, beams, n, parts, tiles;
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

// A key that n of the wave's lanes reach, and no more than n (all that are not 0, if they are fewer): keys differ.
__device__ __forceinline__ uint64_t nth_bound(uint64_t key, int n) {
  if (__popcll(__ballot(key != 0)) <= n) return 1;
  uint64_t at = 0;
#pragma unroll 1
  for (int half = 1; half >= 0; --half) {
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint64_t next = at | 1ull << (32 * half + bit);
      const int reach = __popcll(__ballot(key >= next));
      if (reach >= n) at = next;
      if (reach == n) return at;
    }
  }
  return at;
}

template <typename E>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(BeamArgs a) {
  extern __shared__ uint64_t list[];  // n kept before + kWaves * n * kPer
  __shared__ uint64_t bounds[kWaves], kept[kMostKept];
  __shared__ float red_m[kWaves];
  __shared__ double red_s[kWaves];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long r = blockIdx.y;
  const int part = blockIdx.x, n = a.n;
  uint64_t* out = a.keys + (r * a.parts + part) * n;
  const float score = a.scores[r];
  if (!(score > -INFINITY)) {  // a beam that does not count
    if (tid < n) out[tid] = 0;
    if (tid == 0) a.sums[r * a.parts + part] = make_double2(-INFINITY, 0.);
    return;
  }
  const Row<E> row{static_cast<const E*>(a.logits) + r * a.row_stride, a.V};
  const int t0 = (int)((long long)a.tiles * part / a.parts), t1 = (int)((long long)a.tiles * (part + 1) / a.parts);
  float m = -INFINITY;  // of this wave
  double sum = 0.;      // of this lane, in units of exp(m)
  int have = 0;         // keys in `kept`, descending
  for (int t = t0; t < t1; ++t) {
    typename Row<E>::Raw raw[kVecs];
    const int v0 = t * (kTile / 8) + tid;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) raw[j] = row.fetch(v0 + j * kThreads);
    float x[kVecs][8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      row.read(raw[j], v0 + j * kThreads, x[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[j][e]);
    }
    // the lane's largest, its first place
    uint64_t best = 0;
    if (top > -INFINITY) {
      uint32_t at = 0;
#pragma unroll
      for (int j = kVecs - 1; j >= 0; --j)
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if (x[j][e] == top) at = row.first(v0 + j * kThreads) + e;
      best = (uint64_t)key_of(top) << 32 | ~at;
    }
    const uint32_t high = wave_umax((uint32_t)(best >> 32));
    if (high != 0) {
      const float mt = fmaxf(m, value_of(high));
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += __expf(x[j][e] - mt);
      sum = (mt == m ? sum : sum * (double)__expf(m - mt)) + (double)s;
      m = mt;
    }
    uint64_t bound = nth_bound(best, n);
    if (have == n) bound = max(bound, kept[n - 1] + 1);
    if (lane == 0) bounds[wv] = bound;
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kWaves; ++k) bound = max(bound, bounds[k]);
    if (best >= bound) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint64_t key = (uint64_t)key_of(x[j][e]) << 32 | ~(uint32_t)(row.first(v0 + j * kThreads) + e);
          if (x[j][e] > -INFINITY && key >= bound) list[atomicAdd(&count, 1)] = key;
        }
    }
    __syncthreads();
    const int fresh = count;
    if (fresh > 0) {
      // ranks among the new ones and those kept before (which need not reach the bound)
      uint64_t old = tid < have ? kept[tid] : 0;
      const int all = fresh + have;
      if (tid < have) list[fresh + tid] = old;
      __syncthreads();
      for (int i = tid; i < all; i += kThreads) {
        const uint64_t key = list[i];
        int rank = 0;
        for (int k = 0; k < all; ++k) rank += list[k] > key;
        if (rank < n) kept[rank] = key;
      }
      have = min(all, n);
    }
    __syncthreads();
  }
  if (tid < n) out[tid] = tid < have ? kept[tid] : 0;
  // the waves' sums, in a fixed order
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d, kWave);
  if (lane == 0) {
    red_m[wv] = m;
    red_s[wv] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    float mt = red_m[0];
    for (int k = 1; k < kWaves; ++k) mt = fmaxf(mt, red_m[k]);
    double s = 0.;
    for (int k = 0; k < kWaves; ++k)
      if (red_m[k] > -INFINITY) s += red_s[k] * exp((double)red_m[k] - mt);
    a.sums[r * a.parts + part] = make_double2(mt, s);
  }
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

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(BeamArgs a) {
  extern __shared__ uint64_t lds[];  // [beams][parts][n], then [beams][n]
  __shared__ double base[kMostBeams];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.n, lists = a.beams * a.parts;
  const long long r0 = (long long)blockIdx.x * a.beams;
  uint64_t* best = lds + (size_t)lists * n;
  const uint64_t* keys = a.keys + r0 * a.parts * n;
  for (int i = tid; i < lists * n; i += kMergeThreads) lds[i] = keys[i];
  __syncthreads();
  for (int b = wv; b < a.beams; b += kMergeThreads / kWave) {
    const double2 ms = lane < a.parts ? a.sums[(r0 + b) * a.parts + lane] : make_double2(-INFINITY, 0.);
    const double m = value_of(wave_umax(key_of((float)ms.x)));
    double s = ms.x > -INFINITY ? ms.y * exp(ms.x - m) : 0.;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) s += __shfl_xor(s, d, kWave);
    if (lane == 0) base[b] = (double)fminf(a.scores[r0 + b], FLT_MAX) - (m + log(s));
    // the parts' lists, each descending, a list to a lane
    const uint64_t* mine = lds + ((size_t)b * a.parts + min(lane, a.parts - 1)) * n;
    uint64_t head = lane < a.parts ? mine[0] : 0;
    int at = 0;
    for (int k = 0; k < n; ++k) {
      const int w = wave_best(head);
      const uint64_t key = w < 0 ? 0 : (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(head >> 32), w) << 32 |
                                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, w);
      if (lane == 0) best[b * n + k] = key;
      if (lane == w) head = ++at < n ? mine[at] : 0;
    }
  }
  __syncthreads();
  if (wv != 0) return;
  // the beams' lists, a beam to a lane
  const uint64_t* mine = best + min(lane, a.beams - 1) * n;
  auto total = [&](uint64_t key) { return key ? order_of(base[min(lane, a.beams - 1)] + value_of((uint32_t)(key >> 32))) : 0; };
  uint64_t key = lane < a.beams ? mine[0] : 0, head = total(key);
  int at = 0;
  for (int k = 0; k < n; ++k) {
    const int w = wave_best(head);
    if (w < 0 ? lane == 0 : lane == w) {
      const size_t o = (size_t)blockIdx.x * n + k;
      a.out_scores[o] = w < 0 ? -INFINITY : (float)(base[lane] + value_of((uint32_t)(key >> 32)));
      a.out_tokens[o] = w < 0 ? -1 : (int)~(uint32_t)key;
      a.out_parents[o] = w;
      key = ++at < n && w >= 0 ? mine[at] : 0;
      head = total(key);
    }
  }
}

struct Plan {
  int tiles, parts;
  size_t bytes;
};

bool sizes_ok(int R, int beams, int V, int n) {
  return R > 0 && beams > 0 && beams <= kMostBeams && V > 0 && V <= (1 << 20) && n > 0 && n <= kMostKept &&
         (long long)R * beams <= 65535;
}

Plan make_plan(int R, int beams, int V, int n) {
  Plan p;
  p.tiles = (V + kTile - 1) / kTile;
  const long long rows = (long long)R * beams;
  const int want = (int)std::max(1ll, 2048 / rows);
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
  const size_t list = ((size_t)n + ns::kWaves * n * ns::kPer) * sizeof(uint64_t);  // (up to 33 KB)
  const dim3 grid(p.parts, (unsigned)rows);
  if (fp32)
    hipLaunchKernelGGL((ns::beam_rows_kernel<float>), grid, dim3(ns::kThreads), list, st, a);
  else
    hipLaunchKernelGGL((ns::beam_rows_kernel<uint16_t>), grid, dim3(ns::kThreads), list, st, a);
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
