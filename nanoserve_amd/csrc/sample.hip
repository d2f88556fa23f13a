// Sampling from logits with temperature, top-k, top-p and min-p and a given random number per row
// (gfx950; contract in batch_ops.h). The reference is greedy (python/nanoserve/qwen.py:166-177).
//
// The kept tokens are a beginning of the order by falling logit, so they are those above a cut: a 32-bit
// order-preserving key of the logit, and the index up to which tokens at exactly that key are kept. The row is
// never sorted. It is read up to four times, by several workgroups per row, in launches of their own:
//   max   the largest logit, and that of every tile of 512
//   hist  a histogram, linear in the logit, of counts for top-k and of weights for top-p: 2048 bins over
//         the logits whose weight is not zero. The cut lies in one bin. Not for a top-k of at most as many
//         tokens as there are tiles: its tokens are not below the k-th largest tile maximum.
//   scan  all tokens down to that bin or maximum into a list, if they fit; else the weights of the bins
//         above it, per tile, and the tokens of that bin into the list
//   end   (one workgroup per row) the list sorted in LDS and cut exactly; the draw, from the list or from
//         the tiles' sums and then within one tile
// hist is left out where no row needs it. top-p of a top-k longer than the list takes scan and
// end twice. hist and scan skip tiles whose maximum does not matter to them. A bin with more tokens than
// the list holds (flat rows, rows of few values) is cut by `end` alone, digit by digit of the key: one workgroup reads
// the row five times (three digits, the level tokens, the sums), eight times with both top-k and top-p.
// Measured: one row of 152064 bf16 with top-k 20 and top-p 0.8 16 us (max 3.4, scan 8, end 5: latency); 256 rows of
// 151936 fp32 with settings of their own 160 us, 167 to 174 among other launches (max 25, at 6.3 TB/s, hist 33, scan 39,
// end 21, second scan 22, end 20). Crowded rows of 152064, top-p 0.9, one row and 256: T = 20 280 and 375 us (end alone
// 268), logits of whole numbers 312 and 436, T = 20 with a top-k of a third of the row in fp32 372 and 509; spread
// rows 31 and 148.
//  * Launches, each with little code, and not one kernel with a counter that finds a row's last workgroup:
//    the fences that its data needs between the XCDs' L2 caches cost more (256 rows without a cut 407 us).
//  * Weights exp((l - max) / T) are rounded to multiples of 2^-42 and summed as integers: sums do not
//    depend on their order (LDS and memory atomics are free to run in any), and a border between two
//    tokens moves by no more than about 2^-26 of the largest weight if all 150 000 roundings went one
//    way, 2^-34 as they fall. fp32 weights would be 2^-24 off each in a way that the row shares, enough
//    to change tokens of a flat row. fp64 runs at the fp32 rate on this GPU.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "batch_ops.h"
#include "spans.h"
#include "w4_common.h"
#include "w4_kernels.h"

namespace ns {
namespace {

constexpr int kThreads = 512;
constexpr int kRowWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr int kBinsPer = kBins / kThreads;
constexpr int kList = 2048;
constexpr int kShort = 512;  // a longer list is sorted in more time than the sums of its tokens' tiles take
constexpr uint32_t kRanked = kThreads;  // the longest list that is ordered by rank, an entry per thread
constexpr int kTileVecs = kWave;  // vectors of 8 logits per tile
static_assert((1 << 20) / (8 * kTileVecs) <= kBins, "tiles of the largest vocabulary take the bins' place");
constexpr int kMaxParts = 64;
constexpr uint32_t kKeyMin = 0x007fffffu;  // key of -inf: never drawn

// What a row's scan does: nothing any more; sums of everything from min-p's cut on; the list down to bin
// `cut`; sums above bin `cut` and that bin's list, for top-k or top-p; nothing, for the slow cut.
enum Todo { kFirst, kDone, kSum, kToList, kTopK, kTopP, kSlow };

struct RowState {
  int todo;
  uint32_t cut;
  float from;      // kToList: the least logit of the list
  uint32_t above;  // kTopK: tokens in higher bins
  uint64_t total;  // kToList: the weights that top-p refers to (0: those of the list's first top_k)
  uint64_t need;   // kTopP: what the weights of the bin's first tokens have to reach
};

// Whether the tiles' maxima bound this top-k.
constexpr int kMostTiles = 1024;
__host__ __device__ inline bool tiles_bound(int top_k, int tiles) {
  return top_k <= tiles && tiles <= kMostTiles && top_k <= kList;
}

struct SampleArgs {
  const void* logits;
  long long row_stride;
  const float *u, *temps, *top_ps, *min_ps;
  const int* top_ks;
  int* out;
  float temp, top_p, min_p;
  int top_k, V, tiles, parts;
  int round;  // of scan and end: 0 or 1
  // per row of the batch
  RowState* state;                    // [2]: of each round
  uint64_t *weights, *list, *tile_w;  // [kBins], [2][kList], [tiles]
  uint32_t *counts, *list_n;          // [kBins], [2]
  float *part_max, *tile_max;         // [kMaxParts], [tiles]
};

// Keys: unsigned order = order of the logits; -0 and +0 have the same key.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (0x80000000u | (uint32_t)((int32_t)b >> 31));
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// NaN -> -inf, +inf -> the largest finite value, -0 -> +0
__device__ __forceinline__ float clean(float x) {
  return (x == x ? fminf(x, FLT_MAX) : -INFINITY) + 0.f;
}

// A constant that the compiler holds in a scalar register pair: as a literal it would be copied to vector
// registers before every use (v_fmac_f64 overwrites its addend).
__device__ __forceinline__ double scalar(double c) {
  asm("" : "+s"(c));
  return c;
}

// exp((x - top) / T) in units of 2^-42, rounded to nearest: y = log2 of it in fp64, its nearest integer k
// by adding 1.5 2^52 (k is then the low word), 2^(y - k) by the polynomial of degree 9 that interpolates
// 2^f at the Chebyshev points of [-1/2, 1/2] (off by 2^-45.6 at most), k added to its exponent, and the
// rounding by adding 2^52. Less than half a unit is zero.
struct Weight {
  double top, scale;  // scale = log2(e) / T
  __device__ uint64_t operator()(float x) const {
    constexpr double kUnit = 4398046511104.0, kRound = 6755399441055744.0, kInt = 4503599627370496.0;
    const double y = ((double)x - top) * scale, round = scalar(kRound), t = y + round, f = y - (t - round);
    double p = scalar(1.0205905413765595e-07 * kUnit);
    p = fma(p, f, scalar(1.325964524488711e-06 * kUnit));
    p = fma(p, f, scalar(1.5252672924850737e-05 * kUnit));
    p = fma(p, f, scalar(0.0001540343375125101 * kUnit));
    p = fma(p, f, scalar(0.0013333558200794592 * kUnit));
    p = fma(p, f, scalar(0.009618129193934313 * kUnit));
    p = fma(p, f, scalar(0.05550410866465167 * kUnit));
    p = fma(p, f, scalar(0.2402265069564034 * kUnit));
    p = fma(p, f, scalar(0.6931471805599462 * kUnit));
    p = fma(p, f, scalar(1.0000000000000135 * kUnit));
    const uint64_t b = __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, t) << 52);
    const uint64_t w = __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, b) + scalar(kInt)) -
                       __builtin_bit_cast(uint64_t, kInt);
    return y >= -43.5 ? w : 0;
  }
};

// Inclusive prefix sums over the wave by DPP (row shifts, then row broadcasts), without the LDS round
// trips of lane shuffles.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, false);
}
template <int kCtrl, int kRows>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
  return (uint64_t)dpp<kCtrl, kRows>((uint32_t)(v >> 32)) << 32 | dpp<kCtrl, kRows>((uint32_t)v);
}
template <typename T>
__device__ __forceinline__ T wave_inclusive(T v) {
  v += dpp<0x111, 0xf>(v);
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);
  v += dpp<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
  v = wave_inclusive(v);
  return (uint64_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, 63);
}

// Sum of the values of the threads before this one; `all` is the workgroup's sum. red: one slot per wave.
template <typename T>
__device__ __forceinline__ T block_exclusive(T v, T& all, T* red) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const T incl = wave_inclusive(v);
  __syncthreads();  // red may still be read from the call before
  if (lane == 63) red[wv] = incl;
  __syncthreads();
  T before = 0;
  all = 0;
#pragma unroll
  for (int k = 0; k < kRowWaves; ++k) {
    const T r = red[k];
    before += k < wv ? r : T(0);
    all += r;
  }
  return before + incl - v;
}

// Vector i of a row: logits first(i) .. first(i) + 7, which are 8 i .. except that the last vectors end with
// the row and leave out (as -inf) what is another vector's. Loads (fetch) and their use (read) are apart, so that
// several loads can be in flight, and never leave the row; rows start at any element.
template <typename E>
struct Row {
  const E* p;
  int V;
  struct Raw {
    uint32_t w[2 * sizeof(E)];
  };
  __device__ int first(int i) const { return max(min(8 * i, V - 8), 0); }
  __device__ Raw fetch(int i) const {
    struct __attribute__((packed, aligned(sizeof(E)))) Quad { uint32_t w[4]; };
    Raw r;
    const E* at = p + first(i);
    if (V >= 8) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(E) / 2; ++q) {
        const Quad v = reinterpret_cast<const Quad*>(at)[q];
#pragma unroll
        for (int e = 0; e < 4; ++e) r.w[4 * q + e] = v.w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 2 * (int)sizeof(E); ++e) r.w[e] = 0;
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < V) {
          if constexpr (sizeof(E) == 2)
            r.w[e >> 1] |= (uint32_t)at[e] << 16 * (e & 1);
          else
            r.w[e] = __float_as_uint(at[e]);
        }
    }
    return r;
  }
  __device__ void read(const Raw& r, int i, float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = sizeof(E) == 2 ? r.w[e >> 1] : r.w[e];
      x[e] = clean(__uint_as_float(sizeof(E) == 4 ? w : e & 1 ? w & 0xffff0000u : w << 16));
    }
    if (__any(8 * i + 8 > V)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = first(i) + e;
        x[e] = ((at >= 8 * i) & (at < V)) ? x[e] : -INFINITY;
      }
    }
  }
  __device__ void load(int i, float (&x)[8]) const { read(fetch(i), i, x); }
};

__device__ __forceinline__ float max8(const float (&x)[8]) {
  float m = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
  return m;
}

// f(tile, first index, eight logits) for the tiles t0 .. t1 - 1 whose maximum is wanted, dealt to the waves,
// kAtOnce in flight; left(tile) in one lane for each of the others.
template <int kAtOnce, typename E, class Want, class F, class Left>
__device__ __forceinline__ void each_tile(const Row<E>& row, const float* tile_max, int t0, int t1, Want want, F f,
                                          Left left) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int base = t0 + wv; base < t1; base += kRowWaves * kWave) {
    const int mine = base + kRowWaves * lane;
    const bool in = mine < t1, wanted = in && want(tile_max[min(mine, t1 - 1)]);
    if (in && !wanted) left(mine);
    uint64_t mask = __ballot(wanted);
    while (mask) {
      int t[kAtOnce], n = 0;
      typename Row<E>::Raw raw[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {  // (past the last: the same tile again, unused)
        if (mask) {
          t[u] = base + kRowWaves * __builtin_ctzll(mask);
          mask &= mask - 1;
          ++n;
        } else {
          t[u] = t[u ? u - 1 : 0];
        }
        raw[u] = row.fetch(t[u] * kTileVecs + lane);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (u < n) {
          float x[8];
          const int v = t[u] * kTileVecs + lane;
          row.read(raw[u], v, x);
          f(t[u], row.first(v), x);
        }
    }
  }
}

// One row's settings and what follows from its largest logit.
struct Settings {
  float T, top_p, min_p, u;
  int top_k;
  bool k_on, p_on, m_on, greedy, weighted, by_tiles;
  float top, bins_per, low;  // logits below `low` weigh nothing
  uint32_t min_key;
  Weight weight;

  __device__ Settings(const SampleArgs& a, int r) {
    T = a.temps ? a.temps[r] : a.temp;
    top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    min_p = fminf(a.min_ps ? a.min_ps[r] : a.min_p, 1.f);
    top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    u = a.u[r];
    k_on = top_k > 0 && top_k < a.V;
    p_on = top_p < 1.f;
    m_on = min_p > 0.f;
    greedy = !(T > 0.f) || top_k == 1 || top_p <= 0.f;
    weighted = p_on && (!k_on || top_k > kList);  // else the list has all weights that top-p needs
    by_tiles = k_on && tiles_bound(top_k, a.tiles);
    const int lane = threadIdx.x & 63;
    top = wave_max(lane < a.parts ? a.part_max[r * kMaxParts + lane] : -INFINITY);
    if (top == -INFINITY) greedy = true;
    const double scale = 1.4426950408889634 / (double)T;
    // two keys lower for the conversion to fp32
    const float l = (float)fmax((double)top - 43.5 / scale, -(double)FLT_MAX);
    low = fmaxf(value_of(max(key_of(l), kKeyMin + 3) - 2), -FLT_MAX);
    weight = Weight{(double)top, scale};
    bins_per = fminf((float)(kBins * scale / 43.5), 1e30f);
  }
  // min-p: the smallest key that passes
  __device__ void set_min_key() {
    min_key = 0;
    if (!m_on) return;
    const double least = log((double)min_p) * 1.4426950408889634;
    uint32_t lo = kKeyMin, hi = key_of(top);  // the answer is in (lo, hi]
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (((double)value_of(mid) - weight.top) * weight.scale >= least)
        hi = mid;
      else
        lo = mid;
    }
    min_key = hi;
  }
  // falling with the logit, equal for equal ones
  __device__ uint32_t bin(float x) const { return (uint32_t)fminf((top - x) * bins_per, (float)(kBins - 1)); }
  // the target of the draw among kept weights that add up to `sum`
  __device__ uint64_t draw(uint64_t sum) const {
    const double t = u > 0.f ? (double)u * (double)sum : 0.0;
    const uint64_t v = t < (double)sum ? (uint64_t)t : sum;
    return v < sum ? v : sum - 1;
  }
  // the sum that top-p has to reach, of `sum`
  __device__ uint64_t reach(uint64_t sum) const {
    const double t = ceil((double)sum * (double)top_p);
    return t > 1.0 ? min((uint64_t)t, sum) : 1;
  }
};

struct Scratch {  // of the workgroup-wide sums and searches
  uint64_t red64[kRowWaves], hit64;
  uint32_t red32[kRowWaves], hit, above, in;
};

// The bin, from the first on (last: from the last down), at which the running sum of h reaches `target`
// (at least 1; at most the whole sum counts), and the sum before it.
template <bool kLast, typename T>
__device__ __forceinline__ uint32_t crossing(const T* h, T target, T& before, T* red, Scratch& s) {
  T v[kBinsPer], sum = 0, all;
#pragma unroll
  for (int e = 0; e < kBinsPer; ++e) {
    const int i = kBinsPer * threadIdx.x + e;
    v[e] = h[kLast ? kBins - 1 - i : i];
    sum += v[e];
  }
  T ex = block_exclusive<T>(sum, all, red);
  if (target > all) target = all;
#pragma unroll
  for (int e = 0; e < kBinsPer; ++e) {
    if (ex < target && ex + v[e] >= target) {
      const int i = kBinsPer * threadIdx.x + e;
      s.hit = kLast ? kBins - 1 - i : i;
      s.hit64 = ex;
    }
    ex += v[e];
  }
  __syncthreads();
  before = (T)s.hit64;
  const uint32_t bin = s.hit;
  __syncthreads();
  return bin;
}


// Part `part` of the row's tiles.
__device__ __forceinline__ void part_tiles(const SampleArgs& a, int part, int& t0, int& t1) {
  const int per = (a.tiles + a.parts - 1) / a.parts;
  t0 = min(part * per, a.tiles);
  t1 = min(t0 + per, a.tiles);
}

// ------------------------------------------------------------------ max
// Also clears what the next launches add to.
template <typename E>
__global__ void __launch_bounds__(kThreads) sample_max_kernel(SampleArgs a) {
  __shared__ float red[kRowWaves];
  const int r = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Row<E> row{static_cast<const E*>(a.logits) + (size_t)r * a.row_stride, a.V};
  float* tile_max = a.tile_max + (size_t)r * a.tiles;
  int t0, t1;
  part_tiles(a, part, t0, t1);
  for (int i = part * kThreads + tid; i < kBins; i += a.parts * kThreads) {
    a.weights[(size_t)r * kBins + i] = 0;
    a.counts[(size_t)r * kBins + i] = 0;
  }
  if (part == 0 && tid < 2) {
    a.list_n[2 * r + tid] = 0;
    a.state[2 * r + tid] = RowState{};
  }
  float top = -INFINITY;
  for (int t = t0 + wv; t < t1; t += 4 * kRowWaves) {
    typename Row<E>::Raw raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = row.fetch(min(t + u * kRowWaves, t1 - 1) * kTileVecs + lane);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (t + u * kRowWaves < t1) {
        float x[8];
        row.read(raw[u], (t + u * kRowWaves) * kTileVecs + lane, x);
        const float m = wave_max(max8(x));
        if (lane == 0) tile_max[t + u * kRowWaves] = m;
        top = fmaxf(top, m);
      }
  }
  if (lane == 0) red[wv] = top;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int k = 0; k < kRowWaves; ++k) top = fmaxf(top, red[k]);
    a.part_max[r * kMaxParts + part] = top;
  }
}

// ------------------------------------------------------------------ hist
template <typename E>
__global__ void __launch_bounds__(kThreads, 4) sample_hist_kernel(SampleArgs a) {
  __shared__ uint64_t weights[kBins];
  __shared__ uint32_t counts[kBins];
  const int r = blockIdx.y, tid = threadIdx.x;
  const Settings c(a, r);
  if (c.greedy || c.by_tiles || !(c.k_on || c.p_on)) return;
  const Row<E> row{static_cast<const E*>(a.logits) + (size_t)r * a.row_stride, a.V};
  int t0, t1;
  part_tiles(a, blockIdx.x, t0, t1);
  for (int i = tid; i < kBins; i += kThreads) {
    counts[i] = 0;
    if (c.weighted) weights[i] = 0;
  }
  __syncthreads();
  auto want = [&](float m) { return m >= c.low; };
  const float* tile_max = a.tile_max + (size_t)r * a.tiles;
  if (c.weighted)
    each_tile<2>(row, tile_max, t0, t1, want, [&](int, int, const float (&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] >= c.low) {
          const uint32_t b = c.bin(x[e]);
          atomicAdd(&counts[b], 1u);
          atomicAdd(reinterpret_cast<unsigned long long*>(&weights[b]), (unsigned long long)c.weight(x[e]));
        }
    }, [](int) {});
  else
    each_tile<4>(row, tile_max, t0, t1, want, [&](int, int, const float (&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] >= c.low) atomicAdd(&counts[c.bin(x[e])], 1u);
    }, [](int) {});
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) {
    if (counts[i]) atomicAdd(&a.counts[(size_t)r * kBins + i], counts[i]);
    if (c.weighted && weights[i])
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.weights[(size_t)r * kBins + i]),
                (unsigned long long)weights[i]);
  }
}

// ------------------------------------------------------------------ scan
// A row's tile maxima, dealt to the lanes of each wave.
struct Maxima {
  static constexpr int kPer = kMostTiles / kWave;
  uint32_t key[kPer];
  __device__ Maxima(const float* tile_max, int tiles) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kPer; i += 4)
      if (kWave * i < tiles) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = lane + kWave * (i + e);
          key[i + e] = __float_as_uint(tile_max[min(at, tiles - 1)]);
        }
      }
  }
};
// The k-th largest tile maximum, down to its key's upper bits (for bf16 exactly): the largest value of so many bits that at
// least k maxima reach, two bits at a time. Each wave by itself, the maxima in registers (us, against ranking every
// maximum among all of them in LDS: one row of 152064 with top-k 20 16.7 -> 16.2, of 409600 with top-k 600 49 -> 40).
__device__ __forceinline__ float kth_maximum(Maxima& m, int tiles, int k, int bits) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < Maxima::kPer; ++i)
    if (kWave * (i & ~3) < tiles) m.key[i] = lane + kWave * i < tiles ? key_of(__uint_as_float(m.key[i])) : 0;
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = 30; bit >= 32 - bits; bit -= 2) {
    const uint32_t n1 = t | 1u << bit, n2 = t | 2u << bit, n3 = t | 3u << bit;
    int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
    for (int i = 0; i < Maxima::kPer; i += 4)
      if (kWave * i < tiles) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c1 += __builtin_popcountll(__ballot(m.key[i + e] >= n1));
          c2 += __builtin_popcountll(__ballot(m.key[i + e] >= n2));
          c3 += __builtin_popcountll(__ballot(m.key[i + e] >= n3));
        }
      }
    t = c3 >= k ? n3 : c2 >= k ? n2 : c1 >= k ? n1 : t;
  }
  return value_of(t);  // (NaN where fewer than k are above -inf)
}

// What the row's histogram says.
__device__ __forceinline__ RowState decide(const SampleArgs& a, int r, const Settings& c, Maxima& maxima, int key_bits,
                                          Scratch& s) {
  const int tid = threadIdx.x;
  RowState st{};
  if (c.greedy || !(c.k_on || c.p_on)) {
    st.todo = c.greedy ? kDone : kSum;
    return st;
  }
  st.from = c.low;
  if (c.by_tiles) {
    const float least = kth_maximum(maxima, a.tiles, c.top_k, key_bits);
    st.todo = kToList;
    st.cut = kBins - 1;
    st.from = fmaxf(least, c.low);
    return st;
  }
  // this thread's bins, and the counts and weights of those before them
  uint32_t in[kBinsPer], some = 0, n;
  uint64_t w[kBinsPer], sum = 0, total = 0;
#pragma unroll
  for (int e = 0; e < kBinsPer; ++e) {
    in[e] = a.counts[(size_t)r * kBins + kBinsPer * tid + e];
    w[e] = c.weighted ? a.weights[(size_t)r * kBins + kBinsPer * tid + e] : 0;
    some += in[e];
    sum += w[e];
  }
  uint32_t before = block_exclusive<uint32_t>(some, n, s.red32);
  const bool by_count = c.k_on && (uint32_t)c.top_k < n;
  if (!by_count && (n <= kShort || (c.p_on && !c.weighted))) {  // (without weights n <= top_k <= kList)
    st.cut = kBins - 1;
    st.todo = kToList;
    return st;
  }
  if (!by_count && !c.p_on) {
    st.todo = kSum;
    return st;
  }
  uint64_t done = c.weighted ? block_exclusive<uint64_t>(sum, total, s.red64) : 0;
  const uint64_t need = c.reach(total);
#pragma unroll
  for (int e = 0; e < kBinsPer; ++e) {
    const bool here = by_count ? before < (uint32_t)c.top_k && before + in[e] >= (uint32_t)c.top_k
                               : done < need && done + w[e] >= need;
    if (here) {
      s.hit = kBinsPer * tid + e;
      s.above = before;
      s.in = in[e];
      s.hit64 = done;
    }
    before += in[e];
    done += w[e];
  }
  __syncthreads();
  st.cut = s.hit;
  const uint32_t above = s.above, level = s.in;
  if (by_count) {
    st.above = above;
    st.todo = above + level <= kList ? kToList : c.top_k > kList && level <= kList ? kTopK : kSlow;
  } else {
    st.total = total;
    st.need = need - s.hit64;
    st.todo = above + level <= kShort ? kToList : level <= kList ? kTopP : kSlow;
  }
  return st;
}

template <typename E>
__global__ void __launch_bounds__(kThreads, 4) sample_scan_kernel(SampleArgs a) {
  __shared__ uint64_t list[kList];
  __shared__ Scratch s;
  __shared__ uint32_t n, base;
  const int r = blockIdx.y, tid = threadIdx.x;
  RowState* state = a.state + 2 * r + a.round;
  if (a.round && state->todo == kDone) return;
  Maxima maxima(a.tile_max + (size_t)r * a.tiles, a.tiles <= kMostTiles ? a.tiles : 0);  // (in flight with the settings)
  Settings c(a, r);
  RowState st;
  if (a.round == 0) {
    st = decide(a, r, c, maxima, sizeof(E) == 2 ? 16 : 20, s);
    if (blockIdx.x == 0 && tid == 0) *state = st;
  } else {
    st = *state;
  }
  if (st.todo == kDone || st.todo == kSlow) return;
  if (tid == 0) n = 0;
  __syncthreads();
  const Row<E> row{static_cast<const E*>(a.logits) + (size_t)r * a.row_stride, a.V};
  const float* tile_max = a.tile_max + (size_t)r * a.tiles;
  int t0, t1;
  part_tiles(a, blockIdx.x, t0, t1);
  const float low = c.low;
  const uint32_t cut = st.cut;
  auto put = [&](float x, int index) {
    const uint32_t at = atomicAdd(&n, 1u);
    if (at < kList) list[at] = (uint64_t)~key_of(x) << 32 | (uint32_t)index;
  };
  if (st.todo == kToList) {
    const float from = st.from;
    each_tile<4>(row, tile_max, t0, t1, [&](float m) { return m >= from && c.bin(m) <= cut; },
                 [&](int, int i, const float (&x)[8]) {
#pragma unroll
                   for (int e = 0; e < 8; ++e)
                     if (x[e] >= from && c.bin(x[e]) <= cut) put(x[e], i + e);
                 }, [](int) {});
  } else {
    c.set_min_key();
    uint64_t* tile_w = a.tile_w + (size_t)r * a.tiles;
    auto none = [&](int t) { tile_w[t] = 0; };
    auto store = [&](int t, uint64_t sum) {
      sum = wave_total(sum);
      if ((tid & 63) == 0) tile_w[t] = sum;
    };
    const float least = fmaxf(low, c.min_key > kKeyMin ? value_of(c.min_key) : -FLT_MAX);
    if (st.todo == kSum) {
      each_tile<2>(row, tile_max, t0, t1, [&](float m) { return m >= least; },
                   [&](int t, int, const float (&x)[8]) {
                     uint64_t sum = 0;
#pragma unroll
                     for (int e = 0; e < 8; ++e) sum += x[e] >= least ? c.weight(x[e]) : 0;
                     store(t, sum);
                   }, none);
      return;
    }
    each_tile<2>(row, tile_max, t0, t1, [&](float m) { return m >= low && c.bin(m) <= cut; },
                 [&](int t, int i, const float (&x)[8]) {
                   uint64_t sum = 0;
#pragma unroll
                   for (int e = 0; e < 8; ++e) {
                     const uint32_t b = c.bin(x[e]);
                     const bool kept = (b < cut) & (x[e] >= least);
                     if (__any(kept)) sum += kept ? c.weight(x[e]) : 0;
                     if ((b == cut) & (x[e] >= low)) put(x[e], i + e);
                   }
                   store(t, sum);
                 }, none);
  }
  __syncthreads();
  // (a list by tiles may overflow, where many tokens are level: its count says so)
  const uint32_t mine = n;
  if (mine == 0) return;
  if (tid == 0) base = atomicAdd(&a.list_n[2 * r + a.round], mine);
  __syncthreads();
  for (uint32_t i = tid; i < mine && base + i < kList; i += kThreads)
    a.list[((size_t)r * 2 + a.round) * kList + base + i] = list[i];
}

// ------------------------------------------------------------------ end
struct EndShared {
  uint64_t list[kList];
  uint64_t weights[kBins];  // of the list in order; the histogram's; the tiles'
  uint32_t counts[kBins];
  Scratch s;
  int first;
  uint32_t last;
};

// top-p's bin by the histogram's weights
__device__ __forceinline__ void cut_by_weight(const Settings& c, const uint64_t* weights, const uint32_t* counts,
                                              Scratch& s, RowState& st) {
  uint64_t sum = 0, total, done;
  for (int i = threadIdx.x; i < kBins; i += kThreads) sum += weights[i];
  block_exclusive<uint64_t>(sum, total, s.red64);
  const uint64_t need = c.reach(total);
  st.cut = crossing<false, uint64_t>(weights, need, done, s.red64, s);
  uint32_t some = 0, n;
  for (int i = threadIdx.x; i <= (int)st.cut; i += kThreads) some += counts[i];
  block_exclusive<uint32_t>(some, n, s.red32);
  st.total = total;
  st.from = c.low;
  st.need = need - done;
  st.todo = n <= kShort ? kToList : counts[st.cut] <= kList ? kTopP : kSlow;
}

// Ascending, n2 a power of two. Thread t exchanges pair t: with distances up to 64 a wave's pairs stay
// within its own 128 values, in order by themselves, and only the other steps need the workgroup's barrier
// (2048 values: 14 of 66).
__device__ __forceinline__ void sort_list(uint64_t* v, int n2) {
  __syncthreads();
  bool apart = false;
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j > kWave || apart)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      apart = j > kWave;
      for (int t = threadIdx.x; t < n2 / 2; t += kThreads) {
        const int lo = 2 * (t & ~(j - 1)) + (t & (j - 1)), hi = lo + j;
        const uint64_t a = v[lo], b = v[hi];
        if ((a > b) == ((lo & k) == 0)) {
          v[lo] = b;
          v[hi] = a;
        }
      }
    }
  __syncthreads();
}

// Sorts the list's n entries (key falling, index rising; no two are equal), the entries up to a power of two set aside.
// A short list by rank: an entry's place is the number of those before it, read as broadcasts (us without, with at
// most 256, 512: one row with top-k 20 18.9, 16.6, 16.6; 8 mixed rows 56.5, 52.3, 50.0; 128 with top-p 80.5, 80.4, 76.7).
__device__ __forceinline__ void order_list(EndShared& s, uint32_t n) {
  if (n <= kRanked) {
    const int tid = threadIdx.x;
    if (tid < 4) s.list[n + tid] = ~0ull;
    __syncthreads();
    const bool in = tid < (int)n;
    const uint64_t mine = s.list[in ? tid : 0];
    uint32_t at = 0;
    if (__any(in)) {
      for (uint32_t j = 0; j < n; j += 4) {
        uint64_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = s.list[j + e];
#pragma unroll
        for (int e = 0; e < 4; ++e) at += v[e] < mine;
      }
    }
    __syncthreads();
    if (in) s.list[at] = mine;
    __syncthreads();
    return;
  }
  int n2 = 2;
  while (n2 < (int)n) n2 <<= 1;
  for (int i = threadIdx.x; i < n2; i += kThreads)
    if (i >= (int)n) s.list[i] = ~0ull;
  sort_list(s.list, n2);
}
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return ~(uint32_t)(e >> 32); }

__device__ __forceinline__ bool pick_here(uint64_t before, uint64_t w, uint64_t target) {
  return before <= target && target < before + w;
}

// The draw by the tiles' sums (in s.weights), then token by token in the tile that it falls into. Kept:
// keys above tau, and those at it below index `end`.
template <typename E>
__device__ __forceinline__ void draw_from_tiles(const Row<E>& row, int tiles, const Settings& c, uint32_t tau,
                                                uint32_t end, EndShared& s, int* out) {
  const int tid = threadIdx.x, lane = tid & 63, per = (tiles + kThreads - 1) / kThreads;
  const int from = min(tid * per, tiles), to = min(from + per, tiles);
  uint64_t sum = 0, all;
  for (int t = from; t < to; ++t) sum += s.weights[t];
  uint64_t ex = block_exclusive<uint64_t>(sum, all, s.s.red64);
  const uint64_t target = c.draw(all);
  for (int t = from; t < to; ++t) {
    if (pick_here(ex, s.weights[t], target)) {
      s.first = t;
      s.s.hit64 = ex;
    }
    ex += s.weights[t];
  }
  __syncthreads();
  if (tid >= kWave) return;
  float x[8];
  const int v = s.first * kTileVecs + lane, i = row.first(v);
  row.load(v, x);
  uint64_t w[8], mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t key = key_of(x[e]);
    w[e] = key > tau || (key == tau && (uint32_t)(i + e) < end) ? c.weight(x[e]) : 0;
    mine += w[e];
  }
  ex = s.s.hit64 + wave_inclusive(mine) - mine;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (pick_here(ex, w[e], target)) *out = i + e;
    ex += w[e];
  }
}

// The cut of a row with crowded bins and its draw, by this workgroup alone: histograms over the key's
// digits (11, 11 and 10 bits), of counts for top-k, then of the weights that top-k keeps for top-p.
template <typename E>
__device__ __forceinline__ void slow_row(const Row<E>& row, const float* tile_max, int tiles, const Settings& c,
                                         EndShared& s, int* out) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t tau = 0, ties = 0;
  auto none = [](int) {};
  auto any = [](float) { return true; };
  auto heavy = [&](float m) { return m >= c.low; };
  if (c.k_on) {
    uint32_t pre = 0, above = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const uint32_t mask = level == 2 ? 1023u : 2047u;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) s.counts[i] = 0;
      __syncthreads();
      each_tile<1>(row, tile_max, 0, tiles, any, [&](int, int, const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = key_of(x[e]);
          if ((level == 0 || (level == 1 ? key >> 21 : key >> 10) == pre) && key > kKeyMin)
            atomicAdd(&s.counts[(key >> shift) & mask], 1u);
        }
      }, none);
      __syncthreads();
      uint32_t more;
      const uint32_t bin = crossing<true, uint32_t>(s.counts, (uint32_t)c.top_k - above, more, s.s.red32, s.s);
      above += more;
      pre = level == 0 ? bin : level == 1 ? pre << 11 | bin : pre << 10 | bin;
    }
    tau = pre;
    ties = min((uint32_t)c.top_k - above, s.counts[pre & 1023u]);
  }
  if (c.p_on) {
    uint64_t need = 0, done = 0;
    uint32_t pre = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const uint32_t mask = level == 2 ? 1023u : 2047u;
      auto in = [&](uint32_t key) { return level == 0 || (level == 1 ? key >> 21 : key >> 10) == pre; };
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) s.weights[i] = 0;
      __syncthreads();
      each_tile<1>(row, tile_max, 0, tiles, heavy, [&](int, int, const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key > tau && in(key) && x[e] >= c.low)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[(key >> shift) & mask]),
                      (unsigned long long)c.weight(x[e]));
        }
      }, none);
      if (tid == 0 && ties > 0 && in(tau))  // the tokens at top-k's cut
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[(tau >> shift) & mask]),
                  (unsigned long long)(ties * c.weight(value_of(tau))));
      __syncthreads();
      if (level == 0) {
        uint64_t sum = 0, all;
        for (int i = tid; i < kBins; i += kThreads) sum += s.weights[i];
        block_exclusive<uint64_t>(sum, all, s.s.red64);
        need = c.reach(all);
      }
      uint64_t more;
      const uint32_t bin = crossing<true, uint64_t>(s.weights, need - done, more, s.s.red64, s.s);
      done += more;
      pre = level == 0 ? bin : level == 1 ? pre << 11 | bin : pre << 10 | bin;
    }
    const uint64_t w = c.weight(value_of(pre));  // (not zero: the sum goes past `need` there)
    ties = (uint32_t)((need - done + w - 1) / w);
    tau = pre;
  }
  if (c.min_key > tau) {
    tau = c.min_key - 1;
    ties = 0;
  }
  // the index behind the last token kept at tau: by the tiles' counts, then in its tile
  __syncthreads();
  if (tid == 0) s.last = 0;
  each_tile<1>(row, tile_max, 0, tiles, any, [&](int t, int, const float (&x)[8]) {
    uint32_t at = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) at += key_of(x[e]) == tau;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at += __shfl_xor(at, o, kWave);
    if (lane == 0) s.counts[t] = at;
  }, none);
  __syncthreads();
  if (ties > 0) {
    const int per = (tiles + kThreads - 1) / kThreads, from = min(tid * per, tiles), to = min(from + per, tiles);
    uint32_t sum = 0, all;
    for (int t = from; t < to; ++t) sum += s.counts[t];
    uint32_t ex = block_exclusive<uint32_t>(sum, all, s.s.red32);
    for (int t = from; t < to; ++t) {
      if (ex < ties && ex + s.counts[t] >= ties) {
        s.first = t;
        s.s.hit = ties - ex;
      }
      ex += s.counts[t];
    }
    __syncthreads();
    if (tid < kWave) {
      float x[8];
      const int v = s.first * kTileVecs + lane, i = row.first(v);
      row.load(v, x);
      uint32_t here = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) here += key_of(x[e]) == tau;
      uint32_t nth = wave_inclusive(here) - here;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (key_of(x[e]) == tau && ++nth == s.s.hit) s.last = i + e + 1;
    }
    __syncthreads();
  }
  const uint32_t end = s.last;
  each_tile<1>(row, tile_max, 0, tiles, heavy, [&](int t, int i, const float (&x)[8]) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t key = key_of(x[e]);
      if (key > tau || (key == tau && (uint32_t)(i + e) < end)) sum += c.weight(x[e]);
    }
    sum = wave_total(sum);
    if (lane == 0) s.weights[t] = sum;
  }, [&](int t) { s.weights[t] = 0; });
  __syncthreads();
  draw_from_tiles(row, tiles, c, tau, end, s, out);
}

template <typename E>
__global__ void __launch_bounds__(kThreads) sample_end_kernel(SampleArgs a) {
  __shared__ EndShared s;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RowState st = a.state[2 * r + a.round];
  if (a.round && st.todo == kDone) return;
  // the list's beginning, in flight with the settings; meaningless where there is no list or past its length
  const uint64_t* listed = a.list + ((size_t)r * 2 + a.round) * kList;
  const uint32_t length = a.list_n[2 * r + a.round];
  const uint64_t entry = listed[tid];
  Settings c(a, r);
  const Row<E> row{static_cast<const E*>(a.logits) + (size_t)r * a.row_stride, a.V};
  const float* tile_max = a.tile_max + (size_t)r * a.tiles;
  int* out = a.out + r;
  RowState more{};
  more.todo = kDone;  // what another round has to do
  if (c.greedy) {     // the first of the largest logits
    if (tid == 0) s.first = a.tiles;
    __syncthreads();
    for (int t = tid; t < a.tiles; t += kThreads)
      if (tile_max[t] == c.top) atomicMin(&s.first, t);
    __syncthreads();
    if (tid < kWave) {
      float x[8];
      const int v = s.first * kTileVecs + lane;
      row.load(v, x);
      const uint64_t has = __ballot(max8(x) == c.top);
      if (lane == __builtin_ctzll(has)) {
        int e = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (x[i] == c.top) e = i;
        *out = c.top == -INFINITY ? -1 : row.first(v) + e;
      }
    }
  } else {
    c.set_min_key();
    uint32_t n = 0;
    if (st.todo != kSum && st.todo != kSlow) {
      n = length;
      s.list[tid] = entry;
      for (uint32_t i = tid + kThreads; i < n && n <= kList; i += kThreads) s.list[i] = listed[i];
      __syncthreads();
    }
    if (st.todo == kSlow || n > kList) {
      slow_row(row, tile_max, a.tiles, c, s, out);
    } else {
      // the exact cut in the list: its tokens in order, as many as top-k has left or top-p needs
      constexpr int kPer = kList / kThreads;
      uint32_t keep = 0, tau = 0, end = 0;
      uint64_t w[kPer], sum = 0, all;
      if (st.todo != kSum) {
        order_list(s, n);
        if (st.todo == kTopK)
          keep = min((uint32_t)c.top_k - st.above, n);
        else
          keep = st.todo == kToList && c.k_on ? min((uint32_t)c.top_k, n) : n;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const uint32_t i = kPer * tid + e;
          w[e] = i < keep ? c.weight(value_of(entry_key(s.list[i]))) : 0;
          sum += w[e];
        }
        uint64_t ex = block_exclusive<uint64_t>(sum, all, s.s.red64);
        uint64_t need = st.todo == kTopP ? st.need : c.reach(st.total ? st.total : all);
        bool shorten = c.p_on;
        if (st.todo == kTopK && c.p_on) {
          shorten = false;  // top-p of what top-k keeps: perhaps in another bin
          for (int i = tid; i < kBins; i += kThreads) {
            s.counts[i] = a.counts[(size_t)r * kBins + i];
            s.weights[i] = i < (int)st.cut ? a.weights[(size_t)r * kBins + i] : i == (int)st.cut ? all : 0;
          }
          __syncthreads();
          cut_by_weight(c, s.weights, s.counts, s.s, more);
          if (more.todo != kSlow && more.cut == st.cut) {
            more.todo = kDone;
            need = more.need;
            shorten = true;
          } else if (more.todo == kSlow) {
            more.todo = kDone;
            slow_row(row, tile_max, a.tiles, c, s, out);
            if (tid == 0) a.state[2 * r + 1] = more;
            return;
          }
        }
        if (shorten) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (ex < need && ex + w[e] >= need) s.last = kPer * tid + e;
            ex += w[e];
          }
          __syncthreads();
          keep = s.last + 1;
        }
        tau = entry_key(s.list[keep - 1]);
        end = (uint32_t)s.list[keep - 1] + 1;
      }
      if (st.todo == kToList && keep <= 2 * kWave) {
        // few tokens: each adds up those up to its index
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (kPer * tid + e < keep) s.weights[kPer * tid + e] = entry_key(s.list[kPer * tid + e]) >= c.min_key ? w[e] : 0;
        __syncthreads();
        if (tid < (int)keep) {
          const uint32_t index = (uint32_t)s.list[tid];
          uint64_t upto = 0, whole = 0;
          for (uint32_t j = 0; j < keep; ++j) {
            const uint64_t v = s.weights[j];
            whole += v;
            upto += (uint32_t)s.list[j] <= index ? v : 0;
          }
          const uint64_t v = s.weights[tid];
          if (pick_here(upto - v, v, c.draw(whole))) *out = (int)index;
        }
      } else if (more.todo == kDone) {
        for (int t = tid; t < a.tiles; t += kThreads)
          s.weights[t] = st.todo == kToList ? 0 : a.tile_w[(size_t)r * a.tiles + t];
        __syncthreads();
        // the list's kept tokens join their tiles
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const uint32_t i = kPer * tid + e;
          if (i < keep && entry_key(s.list[i]) >= c.min_key)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[(uint32_t)s.list[i] / (8 * kTileVecs)]),
                      (unsigned long long)w[e]);
        }
        __syncthreads();
        if (c.min_key > tau) {  // everything from min-p's cut on
          tau = c.min_key - 1;
          end = 0;
        }
        draw_from_tiles(row, a.tiles, c, tau, end, s, out);
      }
    }
  }
  if (a.round == 0 && tid == 0) a.state[2 * r + 1] = more;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int row_tiles(int V) { return (V + 8 * kTileVecs - 1) / (8 * kTileVecs); }

// Workgroups per row, each with at least eight tiles: two per CU where all rows have the same settings and end
// together, six where rows have their own, so that the long ones spread. us with two, four, six and eight per CU:
// 128 rows of 152064 with top-k 20 31, 37, 42, 48; 16 with top-p 33, 38, 38, 38; 256 mixed 234, 174, 158, 154, 64
// mixed 95, 85, 91, 93. Settings in device arrays count as the rows' own whatever they hold, and an array of top-k
// with any top-p brings all launches: top-k 20 and top-p 0.8 for every row of 152064 take, as numbers and as arrays, 16.5
// and 21.4 us for one row, 30 and 47 for 128, 39 and 55 for 256.
int row_parts(int B, int V, bool mixed) {
  int cus = 256;  // (a failed query leaves MI355X's count; the launch reports the error)
  if (cached_cu_count(&cus) != hipSuccess || cus <= 0) cus = 256;
  const int want = ((mixed ? 6 : 2) * cus + B - 1) / B;
  return std::max(1, std::min({want, row_tiles(V) / 8, kMaxParts}));
}

// Workspace of one row: states, histograms, lists, maxima and sums of the tiles.
size_t row_bytes(int V) {
  return sizeof(RowState) * 2 + kBins * 12 + 2 * kList * 8 + 8 + kMaxParts * 4 + (size_t)row_tiles(V) * 12;
}

template <typename E>
void launch_sample(SampleArgs a, int B, hipStream_t st) {
  const bool k = a.top_ks || (a.top_k > 0 && a.top_k < a.V), p = a.top_ps || a.top_p < 1.f;
  const bool greedy = !a.temps && !(a.temp > 0.f);
  const dim3 grid(a.parts, B), block(kThreads);
  hipLaunchKernelGGL(sample_max_kernel<E>, grid, block, 0, st, a);
  const bool by_tiles = k && !a.top_ks && tiles_bound(a.top_k, a.tiles);
  if ((k || p) && !greedy && !by_tiles) hipLaunchKernelGGL(sample_hist_kernel<E>, grid, block, 0, st, a);
  const int rounds = k && p && (a.top_ks || a.top_k > kList) ? 2 : 1;
  for (a.round = 0; a.round < rounds; ++a.round) {
    if (!greedy) hipLaunchKernelGGL(sample_scan_kernel<E>, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_end_kernel<E>, dim3(B), block, 0, st, a);
  }
}

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_sample_workspace(int B, int V, int fp32) {
  (void)fp32;
  if (B <= 0 || V <= 0 || V > (1 << 20)) return 0;
  return ns::row_bytes(V) * B;
}

int ns_sample(const void* logits, int fp32, long long row_stride, const float* u, const float* temps,
              float temp, const int* top_ks, int top_k, const float* top_ps, float top_p,
              const float* min_ps, float min_p, int* out, void* work, size_t work_bytes, int B, int V,
              void* stream) {
  if (B <= 0 || B > 65535 || V <= 0 || V > (1 << 20) || row_stride < V) return -2;
  if (!logits || !u || !out) return -2;
  if (!ns::aligned(logits, fp32 ? 4 : 2) || !ns::aligned(u, 4) || !ns::aligned(temps, 4) ||
      !ns::aligned(top_ks, 4) || !ns::aligned(top_ps, 4) || !ns::aligned(min_ps, 4) || !ns::aligned(out, 4))
    return -2;
  if (!work || !ns::aligned(work, 16) || work_bytes < ns_sample_workspace(B, V, fp32)) return -2;
  const size_t elt = fp32 ? 4 : 2, row = 4 * static_cast<size_t>(B);
  const ns::Bytes y = ns::bytes_of(out, row), w = ns::bytes_of(work, ns_sample_workspace(B, V, fp32)),
                  x = ns::rows_of(logits, B, row_stride, V, elt);
  if (!ns::apart(x, y) || !ns::apart(x, w) || !ns::apart(y, w)) return -2;
  for (const void* p : {static_cast<const void*>(u), static_cast<const void*>(temps), static_cast<const void*>(top_ks),
                        static_cast<const void*>(top_ps), static_cast<const void*>(min_ps)})
    if (!ns::apart(w, ns::bytes_of(p, row))) return -2;
  ns::SampleArgs a{logits, row_stride, u, temps, top_ps, min_ps, top_ks, out, temp, top_p, min_p, top_k, V};
  a.tiles = ns::row_tiles(V);
  a.parts = ns::row_parts(B, V, temps || top_ks || top_ps || min_ps);
  const size_t b = static_cast<size_t>(B);
  a.state = static_cast<ns::RowState*>(work);
  a.weights = reinterpret_cast<uint64_t*>(a.state + b * 2);
  a.list = a.weights + b * ns::kBins;
  a.tile_w = a.list + b * 2 * ns::kList;
  a.counts = reinterpret_cast<uint32_t*>(a.tile_w + b * a.tiles);
  a.list_n = a.counts + b * ns::kBins;
  a.part_max = reinterpret_cast<float*>(a.list_n + b * 2);
  a.tile_max = a.part_max + b * ns::kMaxParts;
  const auto st = static_cast<hipStream_t>(stream);
  if (fp32)
    ns::launch_sample<float>(a, B, st);
  else
    ns::launch_sample<uint16_t>(a, B, st);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
