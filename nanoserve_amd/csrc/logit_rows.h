// Rows of logits as the kernels over a vocabulary read them: order keys and vectors of eight.
#pragma once
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "w4_common.h"

namespace ns {
namespace {

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
  __device__ void read(const Raw& r, int i, float (&x)[8]) const { read(r, i, x, clean); }
  template <class Clean>
  __device__ void read(const Raw& r, int i, float (&x)[8], Clean clean) const {
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

}  // namespace
}  // namespace ns
