// What the paged-cache kernels share: the batch's metadata and the pages' addresses (contracts in
// batch_ops.h).
#pragma once
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "spans.h"
#include "w4_common.h"

namespace ns {

// Inclusive sums over the wave by DPP (row shifts, then row broadcasts).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  auto from = [](uint32_t x, auto ctrl, auto rows) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using M = std::integral_constant<int, 0xf>;
  v += from(v, std::integral_constant<int, 0x111>{}, M{});
  v += from(v, std::integral_constant<int, 0x112>{}, M{});
  v += from(v, std::integral_constant<int, 0x114>{}, M{});
  v += from(v, std::integral_constant<int, 0x118>{}, M{});
  v += from(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  return v + from(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
}

struct Batch {
  const int *q_start, *lens, *table;  // q_start null: one token per sequence
  long long table_stride;
  int T, B, width, page_size;

  __device__ int positions(int b) const { return min(max(lens[b], 0), width * page_size); }
  // first token row and token count of sequence b
  __device__ void tokens(int b, int& row0, int& nn) const {
    if (!q_start) {
      row0 = b;
      nn = 1;
      return;
    }
    row0 = min(max(q_start[b], 0), T);
    nn = max(min(max(q_start[b + 1], 0), T) - row0, 0);
  }
  // the sequence whose tokens hold row t, -1 if none does
  __device__ int sequence(int t) const {
    if (!q_start) return t;
    if (t < q_start[0] || t >= q_start[B]) return -1;
    int lo = 0, hi = B;  // q_start[lo] <= t < q_start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (q_start[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  }
};

struct Pools {
  uint16_t *k, *v;
  long long page_stride, head_stride;  // in elements
  int n_pages;
  int size = 2;  // bytes of an element: 1 for a cache in 8 bits, whose addresses k and v hold all the same
};

// The scales of a cache in 8 bits: one byte e, for 2^(e - 127), per 16 rows of a page and head.
struct Scales {
  uint8_t *k, *v;
  long long page_stride, head_stride;
};
constexpr int kScaleRows = 16;
// Of a scale: the least e with t <= 448 * 2^e, between these two (so that every code times its scale is a normal bf16,
// or 0: 2^-9 * 2^-110 and 448 * 2^119). t finite and not negative.
constexpr int kLeastScale = -110, kMostScale = 119;
__device__ __forceinline__ int scale_exponent(float t) {
  const uint32_t b = __float_as_uint(t);  // 448 = 1.75 * 2^8
  return min(max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u), kLeastScale), kMostScale);
}
// Held to e4m3's range, 448 (the conversion would make NaN of what lies past 464); NaN stays.
__device__ __forceinline__ float held448(float x) { return fabsf(x) > 448.f ? copysignf(448.f, x) : x; }

// Host checks common to the entry points.
inline bool batch_ok(const Batch& s, const Pools& p, int Hk, int D) {
  auto al = [](const void* q, uintptr_t n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; };
  if (s.T <= 0 || s.B <= 0 || s.width <= 0 || s.page_size <= 0 || s.page_size % 16 || p.n_pages <= 0)
    return false;
  if ((long long)s.width * s.page_size >= (1ll << 30) || s.table_stride < s.width) return false;
  if (!s.q_start && s.T != s.B) return false;
  if (!s.lens || !s.table || !p.k || !p.v) return false;
  if (!al(s.lens, 4) || !al(s.table, 4) || !al(s.q_start, 4) || !al(p.k, 16) || !al(p.v, 16)) return false;
  const int per16 = 16 / p.size;
  if (p.page_stride % per16 || p.head_stride % per16 || p.page_stride < 0 || p.head_stride < 0) return false;
  // pages and heads do not overlap, whichever of the two is the outer one
  const long long head = (long long)s.page_size * D;
  if ((Hk > 1 && p.head_stride < head) || (p.n_pages > 1 && p.page_stride < head)) return false;
  if (p.page_stride >> 46 || p.head_stride >> 46) return false;  // past any address
  return Hk == 1 || p.n_pages == 1 || (__int128)(Hk - 1) * p.head_stride + head <= p.page_stride ||
         (__int128)(p.n_pages - 1) * p.page_stride + head <= p.head_stride;
}

// The offsets i * page + j * head, |i| <= pages and |j| <= heads, hold one in (lo, hi)? i and j from 0 on with
// `down` false. A stride of a lone page or head is 0.
template <typename W>
inline bool offset_in(W page, W head, long long pages, long long heads, bool down, W lo, W hi) {
  for (long long j = down ? -heads : 0; j <= heads; ++j) {
    const W from = lo - j * head, to = hi - j * head;
    // the first i past `from`
    const W i = pages ? std::max<W>(from / page - (from % page < 0) + 1, down ? -pages : 0) : 0;
    if (i <= pages && from < i * page && i * page < to) return true;
  }
  return false;
}

// The same for a pool's strides, in bytes.
inline bool pool_offset_in(const Pools& p, int Hk, bool down, __int128 lo, __int128 hi) {
  const long long pages = p.n_pages - 1, heads = Hk - 1;
  const long long page = pages ? p.size * p.page_stride : 0, head = heads ? p.size * p.head_stride : 0;
  const __int128 far = (__int128)pages * page + (__int128)heads * head;
  if (lo >= far || hi <= (down ? -far : 0)) return false;  // (where the pools' spans are apart: no loop)
  const __int128 most = (__int128)1 << 60;  // what the loop's values stay within, eight times
  if (far < most && lo > -most && hi < most) return offset_in<long long>(page, head, pages, heads, down, lo, hi);
  return offset_in<__int128>(page, head, pages, heads, down, lo, hi);
}

// Whether none of the pool's pages lies in a range.
inline bool pool_apart(const uint16_t* pool, const Pools& p, int Hk, long long head, Bytes x) {
  const __int128 from = (__int128)x.lo - reinterpret_cast<uintptr_t>(pool), size = p.size * (__int128)head;
  return x.lo >= x.hi || !pool_offset_in(p, Hk, false, from - size, from + (x.hi - x.lo));
}

inline Bytes lens_of(const Batch& s) { return bytes_of(s.lens, 4 * (size_t)s.B); }
inline Bytes starts_of(const Batch& s) { return bytes_of(s.q_start, 4 * ((size_t)s.B + 1)); }
inline Bytes table_of(const Batch& s) { return rows_of(s.table, s.B, s.table_stride, s.width, 4); }
// What a call writes (x) against the batch's metadata.
inline bool metadata_apart(const Batch& s, Bytes x) {
  return apart(x, lens_of(s)) && apart(x, starts_of(s)) && apart(x, table_of(s));
}

// Whether K and V share no element: a page of V starts less than a page before or behind one of K nowhere.
inline bool pools_apart(const Pools& p, int Hk, long long head) {
  const __int128 d = (__int128)reinterpret_cast<uintptr_t>(p.v) - reinterpret_cast<uintptr_t>(p.k),
                 size = p.size * (__int128)head;
  return !pool_offset_in(p, Hk, true, d - size, d + size);
}

// Host checks of the scales that go with a pool: strides by which pages and heads do not overlap.
inline bool scales_ok(const Scales& f, const Pools& p, int Hk, int page_size) {
  const long long head = page_size / kScaleRows;
  if (!f.k || !f.v || f.page_stride < 0 || f.head_stride < 0 || f.page_stride >> 46 || f.head_stride >> 46) return false;
  if ((Hk > 1 && f.head_stride < head) || (p.n_pages > 1 && f.page_stride < head)) return false;
  return Hk == 1 || p.n_pages == 1 || (__int128)(Hk - 1) * f.head_stride + head <= f.page_stride ||
         (__int128)(p.n_pages - 1) * f.page_stride + head <= f.head_stride;
}

// The scales as pools of one byte per element, for the checks above.
inline Pools scale_pools(const Scales& f, int n_pages) {
  return Pools{reinterpret_cast<uint16_t*>(f.k), reinterpret_cast<uint16_t*>(f.v), f.page_stride, f.head_stride, n_pages, 1};
}

// Pieces of `size` bytes at all sums of a stride times a number below its count (in bytes, none negative).
struct Pieces {
  long long stride[3], count[3];
  long long size;
  __int128 span() const {
    __int128 s = size;
    for (int i = 0; i < 3; ++i) s += (__int128)stride[i] * (count[i] - 1);
    return s;
  }
};

// Whether the pieces of a and those of b, `d` bytes further on, share no byte. Dimensions of the same stride in both, within
// which the others stay, are taken out one by one (a shift of either set by a multiple of the stride meets the same
// pieces); what is left, the heads as a rule, is compared piece by piece, and counts as not apart where that are more than
// 2^20 comparisons.
inline bool pieces_apart(Pieces a, Pieces b, __int128 d) {
  const __int128 sa = a.span(), sb = b.span();
  if (d >= sa || -d >= sb) return true;
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j) {
      const long long s = a.stride[i];
      if (a.count[i] == 1 || s != b.stride[j]) continue;
      const __int128 na = a.count[i], nb = b.count[j];
      if (sa - (na - 1) * s > s || sb - (nb - 1) * s > s) continue;
      Pieces p = a, q = b;
      p.count[i] = q.count[j] = 1;
      __int128 r = d % s;
      if (r < 0) r += s;
      for (const __int128 at : {r, r - s}) {
        const __int128 k = (at - d) / s;  // b's number less a's, where the two lie `at` apart
        if (k > -na && k < nb && !pieces_apart(p, q, at)) return false;
      }
      return true;
    }
  double work = 1;
  for (int i = 0; i < 3; ++i) work *= (double)a.count[i] * (double)b.count[i];
  if (work > (1 << 20)) return false;
  for (long long i0 = 0; i0 < a.count[0]; ++i0)
    for (long long i1 = 0; i1 < a.count[1]; ++i1)
      for (long long i2 = 0; i2 < a.count[2]; ++i2) {
        const __int128 at = (__int128)i0 * a.stride[0] + (__int128)i1 * a.stride[1] + (__int128)i2 * a.stride[2];
        for (long long j0 = 0; j0 < b.count[0]; ++j0)
          for (long long j1 = 0; j1 < b.count[1]; ++j1)
            for (long long j2 = 0; j2 < b.count[2]; ++j2) {
              const __int128 e = d - at + (__int128)j0 * b.stride[0] + (__int128)j1 * b.stride[1] + (__int128)j2 * b.stride[2];
              if (e < a.size && -e < b.size) return false;
            }
      }
  return true;
}

// Whether a pool's pages (heads of `x` bytes) and another's (of `y`) share no byte. Exact where pages are equally far
// apart in both; else their spans have to be apart.
inline bool sets_apart(const void* a, const Pools& p, long long x, const void* b, const Pools& r, long long y, int Hk) {
  auto of = [&](const Pools& q, long long size) {
    return Pieces{{q.size * q.page_stride, q.size * q.head_stride, 0}, {q.n_pages, Hk, 1}, size};
  };
  const Pieces f = of(p, x), g = of(r, y);
  const __int128 d = (__int128)reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a);
  if (d >= f.span() || -d >= g.span()) return true;
  return (p.n_pages == 1 || f.stride[0] == g.stride[0]) && pieces_apart(f, g, d);
}

}  // namespace ns
