// What the paged-cache kernels share: the batch's metadata and the pages' addresses (contracts in
// batch_ops.h).
#pragma once
#include <stdint.h>

#include <algorithm>

#include "spans.h"
#include "w4_common.h"

namespace ns {

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
  long long page_stride, head_stride;
  int n_pages;
};

// Host checks common to the entry points.
inline bool batch_ok(const Batch& s, const Pools& p, int Hk, int D) {
  auto al = [](const void* q, uintptr_t n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; };
  if (s.T <= 0 || s.B <= 0 || s.width <= 0 || s.page_size <= 0 || s.page_size % 16 || p.n_pages <= 0)
    return false;
  if ((long long)s.width * s.page_size >= (1ll << 30) || s.table_stride < s.width) return false;
  if (!s.q_start && s.T != s.B) return false;
  if (!s.lens || !s.table || !p.k || !p.v) return false;
  if (!al(s.lens, 4) || !al(s.table, 4) || !al(s.q_start, 4) || !al(p.k, 16) || !al(p.v, 16)) return false;
  if (p.page_stride % 8 || p.head_stride % 8 || p.page_stride < 0 || p.head_stride < 0) return false;
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
  const long long page = pages ? 2 * p.page_stride : 0, head = heads ? 2 * p.head_stride : 0;
  const __int128 far = (__int128)pages * page + (__int128)heads * head;
  if (lo >= far || hi <= (down ? -far : 0)) return false;  // (where the pools' spans are apart: no loop)
  const __int128 most = (__int128)1 << 60;  // what the loop's values stay within, eight times
  if (far < most && lo > -most && hi < most) return offset_in<long long>(page, head, pages, heads, down, lo, hi);
  return offset_in<__int128>(page, head, pages, heads, down, lo, hi);
}

// Whether none of the pool's pages lies in a range.
inline bool pool_apart(const uint16_t* pool, const Pools& p, int Hk, long long head, Bytes x) {
  const __int128 from = (__int128)x.lo - reinterpret_cast<uintptr_t>(pool), size = 2 * (__int128)head;
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
                 size = 2 * (__int128)head;
  return !pool_offset_in(p, Hk, true, d - size, d + size);
}

}  // namespace ns
