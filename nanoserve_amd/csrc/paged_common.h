// What the paged-cache kernels share: the batch's metadata and the pages' addresses (contracts in
// batch_ops.h).
#pragma once
#include <stdint.h>

#include <algorithm>

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

}  // namespace ns
