// Sampling from logits with temperature, top-k, top-p and min-p and a given random number per row
// (gfx950; contract in batch_ops.h). The reference is greedy (python/nanoserve/qwen.py:166-177).
//
// One workgroup of 16 waves per row. The kept tokens are a beginning of the order by falling logit, so
// they are those above a cut: a 32-bit order-preserving key of the logit, and how many of the tokens at
// exactly that key (the first ones by index). The cut is found by histograms over digits of the key
// (11, 11 and 10 bits), of counts for top-k and of weights for top-p, and never by sorting the row;
// what passes the first digit's cut is mostly short enough for a list in LDS, which is sorted.
//  * Weights exp((l - max) / T) are rounded to multiples of 2^-42 and summed as integers: sums do not
//    depend on their order (LDS atomics are free to run in any), and a border between two tokens moves
//    by no more than about 2^-33 of the sum at 150 000 tokens. fp32 weights would move it by 2^-24 of
//    the largest ones, enough to change tokens of a flat row. fp64 runs at the fp32 rate on this GPU.
//  * Bound by VALU work where every token's weight is needed (about 30 instructions each), by the
//    passes over the row otherwise.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "batch_ops.h"
#include "w4_common.h"

namespace ns {
namespace {

constexpr int kThreads = 1024;
constexpr int kRowWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr int kList = 2048;
constexpr uint32_t kKeyMin = 0x007fffffu;  // key of -inf: never drawn

struct SampleArgs {
  const void* logits;
  long long row_stride;
  const float *u, *temps, *top_ps, *min_ps;
  const int* top_ks;
  int* out;
  float temp, top_p, min_p;
  int top_k, V;
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

// exp((x - top) / T) in units of 2^-42, rounded to nearest: 2^f for |f| <= 1/2 by its Taylor series up
// to degree 11 (the rest is below 2^-47), and the rounding by adding 2^52.
struct Weight {
  double top, scale;  // scale = log2(e) / T
  __device__ uint64_t operator()(float x) const {
    double y = ((double)x - top) * scale;
    y = fmax(y, -1000.0);
    const double k = rint(y), f = (y - k) * 0.6931471805599453;
    double p = 1.0 / 39916800;
    p = fma(p, f, 1.0 / 3628800);
    p = fma(p, f, 1.0 / 362880);
    p = fma(p, f, 1.0 / 40320);
    p = fma(p, f, 1.0 / 5040);
    p = fma(p, f, 1.0 / 720);
    p = fma(p, f, 1.0 / 120);
    p = fma(p, f, 1.0 / 24);
    p = fma(p, f, 1.0 / 6);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    const double t = ldexp(p, (int)k + 42) + 4503599627370496.0;
    return __builtin_bit_cast(uint64_t, t) - 0x4330000000000000ull;
  }
  // whether a weight can be other than zero (2^-43 and more)
  __device__ bool counts(float x) const { return ((double)x - top) * scale >= -43.5; }
};

template <typename T>
__device__ __forceinline__ T wave_inclusive(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const T u = __shfl_up(v, o, kWave);
    v += lane >= o ? u : T(0);
  }
  return v;
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

// Eight neighbouring logits; past the row's end -inf.
struct Row16 {
  const uint16_t* p;
  int V;
  __device__ void load(int i, float (&x)[8]) const {
    struct __attribute__((packed, aligned(2))) Vec { uint32_t w[4]; };
    if (8 * i + 8 <= V) {
      const Vec v = *reinterpret_cast<const Vec*>(p + 8 * (size_t)i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = clean(__uint_as_float(v.w[e] << 16));
        x[2 * e + 1] = clean(__uint_as_float(v.w[e] & 0xffff0000u));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = 8 * i + e < V ? clean(__uint_as_float((uint32_t)p[8 * (size_t)i + e] << 16)) : -INFINITY;
    }
  }
};
struct Row32 {
  const float* p;
  int V;
  __device__ void load(int i, float (&x)[8]) const {
    struct __attribute__((packed, aligned(4))) Vec { float w[4]; };
    if (8 * i + 8 <= V) {
      const Vec a = *reinterpret_cast<const Vec*>(p + 8 * (size_t)i);
      const Vec b = *reinterpret_cast<const Vec*>(p + 8 * (size_t)i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = clean(a.w[e]);
        x[4 + e] = clean(b.w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 8 * i + e < V ? clean(p[8 * (size_t)i + e]) : -INFINITY;
    }
  }
};

// f(first index, eight logits) over the vectors from .. to - 1 of the row, `step` apart, four in flight
template <class Row, class F>
__device__ __forceinline__ void each(const Row& row, int from, int to, int step, F f) {
  for (int i = from; i < to; i += 4 * step) {
    float x[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u * step < to)
        row.load(i + u * step, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * step < to) f(8 * (i + u * step), x[u]);
  }
}

struct Shared {
  uint64_t weights[kBins];  // weights per digit, later those of the list
  uint64_t list[kList];
  uint32_t counts[kBins];
  uint64_t red64[kRowWaves];
  uint32_t red32[kRowWaves];
  uint64_t hit64;
  uint32_t hit, n;
  int first;
};

__device__ __forceinline__ void sort_list(uint64_t* v, int n2) {  // ascending, n2 a power of two
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      const int t = threadIdx.x;
      if (t < n2 / 2) {
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

// The digit, from the highest down, at which the running sum of h reaches `target` (>= 1), and the sum
// before it; the last digit if it never does.
template <typename T>
__device__ __forceinline__ uint32_t crossing(const T* h, T target, T& before, T* red, Shared& s) {
  const int t = threadIdx.x;
  const T a = h[kBins - 1 - 2 * t], b = h[kBins - 2 - 2 * t];
  T all;
  const T ex = block_exclusive<T>(a + b, all, red);
  if (target > all) target = all;
  if (ex < target && ex + a >= target) {
    s.hit = kBins - 1 - 2 * t;
    s.hit64 = ex;
  } else if (ex + a < target && ex + a + b >= target) {
    s.hit = kBins - 2 - 2 * t;
    s.hit64 = ex + a;
  }
  __syncthreads();
  before = (T)s.hit64;
  const uint32_t bin = s.hit;
  __syncthreads();
  return bin;
}

__device__ __forceinline__ bool pick_here(uint64_t before, uint64_t w, uint64_t target) {
  return before <= target && target < before + w;
}

template <class Row, typename E>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const Row row{static_cast<const E*>(a.logits) + (size_t)r * a.row_stride, a.V};
  const int nv = (a.V + 7) / 8;
  const float T = a.temps ? a.temps[r] : a.temp;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  const float min_p = fminf(a.min_ps ? a.min_ps[r] : a.min_p, 1.f);
  const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  const bool k_on = top_k > 0 && top_k < a.V, p_on = top_p < 1.f, m_on = min_p > 0.f;
  const bool greedy = !(T > 0.f) || top_k == 1 || top_p <= 0.f;
  const bool cut = !greedy && (k_on || p_on || m_on);

  // ---- the largest logit, its first vector, and how many logits have each first digit
  for (int i = tid; i < kBins; i += kThreads) s.counts[i] = 0;
  if (tid == 0) s.first = nv;
  __syncthreads();
  float best = -INFINITY;
  int at = nv;
  each(row, tid, nv, kThreads, [&](int i, const float (&x)[8]) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
    if (m > best) {
      best = m;
      at = i >> 3;
    }
    if (cut) {
#pragma unroll
      for (int e = 0; e < 8; ++e) atomicAdd(&s.counts[key_of(x[e]) >> 21], 1u);
    }
  });
  float top = best;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  if (lane == 0) s.red32[wv] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRowWaves; ++k) top = fmaxf(top, __uint_as_float(s.red32[k]));
  if (top == -INFINITY) {
    if (tid == 0) a.out[r] = -1;
    return;
  }
  if (greedy) {
    if (best == top) atomicMin(&s.first, at);
    __syncthreads();
    if (tid == 0) {
      float x[8];
      row.load(s.first, x);
      int e = 0;
      while (x[e] != top) ++e;
      a.out[r] = 8 * s.first + e;
    }
    return;
  }
  const Weight weight{(double)top, 1.4426950408889634 / (double)T};
  const float uu = a.u[r];
  // the target of the draw among kept weights that add up to `sum`
  auto draw = [&](uint64_t sum) {
    const double t = uu > 0.f ? (double)uu * (double)sum : 0.0;
    const uint64_t v = t < (double)sum ? (uint64_t)t : sum;
    return v < sum ? v : sum - 1;
  };

  // ---- min-p: the smallest key that passes
  uint32_t min_key = 0;
  if (m_on) {
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

  // ---- top-k: the first digit of its cut
  uint32_t k_bin = 0, above = 0;  // above: logits with a higher digit
  if (k_on) k_bin = crossing<uint32_t>(s.counts, (uint32_t)top_k, above, s.red32, s);

  // The logits whose first digit is `bin` or more, if they fit the list: sorted, cut exactly, drawn.
  // `total`: the weights top-p refers to (0: those of the list's first top_k). Uniform result.
  auto by_list = [&](uint32_t bin, uint64_t total) {
    uint32_t c = 0;
    for (int i = tid; i < kBins; i += kThreads) c += (uint32_t)i >= bin ? s.counts[i] : 0u;
    uint32_t n;
    block_exclusive<uint32_t>(c, n, s.red32);
    if (n > kList) return false;
    if (tid == 0) s.n = 0;
    __syncthreads();
    each(row, tid, nv, kThreads, [&](int i, const float (&x)[8]) {
      float m = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
      if (key_of(m) >> 21 >= bin) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key >> 21 >= bin && i + e < a.V)
            s.list[atomicAdd(&s.n, 1u)] = (uint64_t)~key << 32 | (uint32_t)(i + e);
        }
      }
    });
    __syncthreads();
    n = s.n;
    int n2 = 2;
    while (n2 < (int)n) n2 <<= 1;
    for (int i = tid; i < n2; i += kThreads)
      if (i >= (int)n) s.list[i] = ~0ull;
    sort_list(s.list, n2);
    if (k_on) n = min(n, (uint32_t)top_k);
    // weights in order, two per thread
    uint64_t w[2], all;
    uint32_t keys[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      keys[e] = i < n ? ~(uint32_t)(s.list[i] >> 32) : 0u;
      w[e] = i < n ? weight(value_of(keys[e])) : 0;
      s.weights[i] = w[e];
    }
    uint64_t ex = block_exclusive<uint64_t>(w[0] + w[1], all, s.red64);
    const double reach = p_on ? ceil((double)(total ? total : all) * (double)top_p) : 0.0;
    const uint64_t need = reach > 1.0 ? (uint64_t)reach : 1;
    uint32_t kept = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      kept += i < n && (i == 0 || ((!p_on || ex < need) && keys[e] >= min_key && keys[e] > kKeyMin));
      ex += w[e];
    }
    uint32_t m;
    block_exclusive<uint32_t>(kept, m, s.red32);
    // the kept ones by index
    uint64_t mine[2];
    n2 = 2;
    while (n2 < (int)m) n2 <<= 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      mine[e] = i < m ? (uint64_t)(uint32_t)s.list[i] << 32 | i : ~0ull;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) s.list[2 * tid + e] = mine[e];
    sort_list(s.list, n2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = 2 * tid + e;
      w[e] = i < m ? s.weights[(uint32_t)s.list[i]] : 0;
    }
    ex = block_exclusive<uint64_t>(w[0] + w[1], all, s.red64);
    const uint64_t target = draw(all);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (pick_here(ex, w[e], target)) a.out[r] = (int)(s.list[2 * tid + e] >> 32);
      ex += w[e];
    }
    return true;
  };
  const uint32_t min_bin = min_key >> 21;
  // (top-p refers to all that top-k keeps, min-p's cut must not shorten the list then)
  if (cut && (k_on || !p_on) && by_list(p_on ? k_bin : max(k_bin, min_bin), 0)) return;

  // ---- the cut: keys above `tau`, and the first `ties` logits (by index) at it
  uint32_t tau = 0, ties = 0;
  // top-k exactly: the second and third digit
  if (k_on) {
    uint32_t pre = k_bin;
#pragma unroll 1
    for (int level = 1; level < 3; ++level) {
      const int shift = level == 1 ? 10 : 0;
      const uint32_t mask = level == 1 ? 2047u : 1023u;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) s.weights[i] = 0;
      __syncthreads();
      uint32_t* h = reinterpret_cast<uint32_t*>(s.weights);
      each(row, tid, nv, kThreads, [&](int, const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = key_of(x[e]);
          if ((level == 1 ? key >> 21 : key >> 10) == pre) atomicAdd(&h[(key >> shift) & mask], 1u);
        }
      });
      __syncthreads();
      uint32_t more;
      const uint32_t bin = crossing<uint32_t>(h, (uint32_t)top_k - above, more, s.red32, s);
      above += more;
      pre = level == 1 ? pre << 11 | bin : pre << 10 | bin;
    }
    tau = pre;
    ties = (uint32_t)top_k - above;
  }
  // top-p: weights per digit of what top-k kept
  if (p_on) {
    uint64_t total = 0, need = 0, done = 0;
    uint32_t pre = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const uint32_t mask = level == 2 ? 1023u : 2047u;
      auto in = [&](uint32_t key) { return level == 0 || (level == 1 ? key >> 21 : key >> 10) == pre; };
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) s.weights[i] = 0;
      __syncthreads();
      each(row, tid, nv, kThreads, [&](int, const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key > tau && in(key) && weight.counts(x[e]))
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[(key >> shift) & mask]),
                      (unsigned long long)weight(x[e]));
        }
      });
      if (tid == 0 && ties > 0 && in(tau))  // the tokens at top-k's cut
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[(tau >> shift) & mask]),
                  (unsigned long long)(ties * weight(value_of(tau))));
      __syncthreads();
      if (level == 0) {
        uint64_t c = s.weights[tid] + s.weights[tid + kThreads];
        block_exclusive<uint64_t>(c, total, s.red64);
        const double reach = ceil((double)total * (double)top_p);
        need = reach > 1.0 ? (uint64_t)reach : 1;
        if (need > total) need = total;
      }
      uint64_t more;
      const uint32_t bin = crossing<uint64_t>(s.weights, need - done, more, s.red64, s);
      done += more;
      pre = level == 0 ? bin : level == 1 ? pre << 11 | bin : pre << 10 | bin;
      if (level == 0 && !k_on && by_list(max(bin, min_bin), total)) return;
    }
    const uint64_t w = weight(value_of(pre));
    ties = (uint32_t)((need - done + w - 1) / w);
    tau = pre;
  }
  if (min_key > tau) {
    tau = min_key - 1;
    ties = 0;
  }

  // ---- the draw: each wave sums the kept weights of its part of the row, then the part that the
  // target falls into is summed vector by vector
  const int part = (nv + kRowWaves - 1) / kRowWaves;
  uint64_t sum = 0;
  uint32_t level = 0;  // tokens at the cut
  each(row, wv * part + lane, min((wv + 1) * part, nv), kWave, [&](int, const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t key = key_of(x[e]);
      level += key == tau;
      if (key > tau && weight.counts(x[e])) sum += weight(x[e]);
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, kWave);
    level += __shfl_xor(level, o, kWave);
  }
  __syncthreads();
  if (lane == 0) {
    s.red64[wv] = sum;
    s.red32[wv] = level;
  }
  __syncthreads();
  const uint64_t wt = ties > 0 ? weight(value_of(tau)) : 0;
  uint64_t all = 0;
  uint32_t left = ties;
#pragma unroll
  for (int k = 0; k < kRowWaves; ++k) {
    const uint32_t c = min(left, s.red32[k]);
    left -= c;
    all += s.red64[k] + c * wt;
  }
  const uint64_t target = draw(all);
  uint64_t before = 0;
  int hit = 0;
  left = ties;
  for (; hit < kRowWaves - 1; ++hit) {
    const uint32_t c = min(left, s.red32[hit]);
    const uint64_t w = s.red64[hit] + c * wt;
    if (target < before + w) break;
    left -= c;
    before += w;
  }
  const int end = min((hit + 1) * part, nv);
  for (int v0 = hit * part; v0 < end; v0 += kThreads) {
    const int v = v0 + tid;
    float x[8];
    uint32_t here = 0;
    uint64_t mine = 0;
    if (v < end) {
      row.load(v, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) here += key_of(x[e]) == tau;
    }
    uint32_t all_ties;
    const uint32_t ex_ties = block_exclusive<uint32_t>(here, all_ties, s.red32);
    uint32_t mine_left = left - min(left, ex_ties);
    uint64_t w[8];
    if (v < end) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = key_of(x[e]);
        const bool tie = key == tau && mine_left > 0;
        mine_left -= tie;
        w[e] = key > tau || tie ? weight(x[e]) : 0;
        mine += w[e];
      }
    }
    uint64_t round;
    uint64_t ex = before + block_exclusive<uint64_t>(mine, round, s.red64);
    if (v < end) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (pick_here(ex, w[e], target)) a.out[r] = 8 * v + e;
        ex += w[e];
      }
    }
    before += round;
    left -= min(left, all_ties);
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_sample_workspace(int, int, int) { return 0; }

int ns_sample(const void* logits, int fp32, long long row_stride, const float* u, const float* temps,
              float temp, const int* top_ks, int top_k, const float* top_ps, float top_p,
              const float* min_ps, float min_p, int* out, void* work, size_t work_bytes, int B, int V,
              void* stream) {
  if (B <= 0 || V <= 0 || V > (1 << 20) || row_stride < V) return -2;
  if (!logits || !u || !out) return -2;
  if (!ns::aligned(logits, fp32 ? 4 : 2) || !ns::aligned(u, 4) || !ns::aligned(temps, 4) ||
      !ns::aligned(top_ks, 4) || !ns::aligned(top_ps, 4) || !ns::aligned(min_ps, 4) || !ns::aligned(out, 4))
    return -2;
  const ns::SampleArgs a{logits, row_stride, u, temps, top_ps, min_ps, top_ks, out,
                         temp, top_p, min_p, top_k, V};
  const auto st = static_cast<hipStream_t>(stream);
  if (fp32)
    hipLaunchKernelGGL((ns::sample_kernel<ns::Row32, float>), dim3(B), dim3(ns::kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((ns::sample_kernel<ns::Row16, uint16_t>), dim3(B), dim3(ns::kThreads), 0, st, a);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
