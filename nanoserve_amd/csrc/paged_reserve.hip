// Block tables, first rows and slot map of a step from its sequences' new lengths (gfx950; contract in batch_ops.h). The
// reference serves one sequence with one cache and has no counterpart.
//
// Prefix sums over the sequences say which free page is whose: page k that the call takes is the k-th from the stack's
// top, so the table entries need no atomics and do not depend on any order. One workgroup does all of it: a call moves a few
// KiB and is bound by the latency of its chain (lengths -> sums -> free pages -> entries -> slots), which a
// second launch would lengthen. Only slot maps of long prompts go to a launch of their own, over many
// workgroups, behind it. Measured: 64 sequences that give back or take drafts 4.6 us, 1000 7.7; 48 prompts of 150 000
// tokens (9500 pages) 10.3 and 4.2 for the slot map. The workgroup's own instructions count: 512 and 256 threads are faster for 64
// sequences (4.1, 3.9) and take 18 and 29 us for the prompts; four entries of a thread at a time 17 for two small calls (9.2).
#include <stdint.h>

#include <algorithm>
#include <iterator>

#include "batch_ops.h"
#include "paged_common.h"

namespace ns {
namespace {

constexpr int kThreads = 1024;

struct ReserveArgs {
  const int* add;
  int *lens, *table, *free, *n_free, *q_start, *shorts;
  long long* slots;
  long long table_stride, capacity;
  int B, width, page_size, rows;  // rows -1: no slot map
};

// Slot maps of more rows have a launch of their own. us of giving back and taking with a launch from 2048 rows on, from 4096
// and from 8192: 2400 rows 13.7, 12.2, 12.2; 6800 13.8, 13.7, 14.6.
constexpr int kOwnRows = 4096;

// What one sequence asks for.
struct Ask {
  int had, has;         // table entries before and after
  int len, grown;       // positions after, new tokens
  bool fits;
  __device__ long long taken() const { return max(has - had, 0); }
  __device__ long long given() const { return max(had - has, 0); }
};

__device__ __forceinline__ Ask ask_of(const ReserveArgs& a, int b) {
  Ask x{0, 0, 0, 0, true};
  if (b >= a.B) return x;
  const long long most = (long long)a.width * a.page_size;
  const long long old = min((long long)max(a.lens[b], 0), most);
  const long long len = max(old + a.add[b], 0ll);
  x.fits = len <= most;
  x.len = (int)min(len, most);
  x.grown = x.fits ? max(a.add[b], 0) : 0;  // (below 2^30)
  x.had = (int)((old + a.page_size - 1) / a.page_size);
  x.has = (int)((x.len + a.page_size - 1) / a.page_size);
  return x;
}

// The slot of a new token of sequence b, `past` positions before its end.
__device__ __forceinline__ long long slot_of(const ReserveArgs& a, int b, int len, int past) {
  const int pos = len - past;
  const int page = a.table[(size_t)b * a.table_stride + pos / a.page_size];
  return page < 0 ? -1 : (long long)page * a.page_size + pos % a.page_size;
}

__global__ void __launch_bounds__(kThreads) reserve_kernel(ReserveArgs a, int with_slots) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ long long part[3][kWaves];
  // per sequence of a chunk: pages taken, pages given, token rows, up to its own (of a call that goes through: below 2^31)
  __shared__ int ends[3][kThreads];
  __shared__ int firsts[2][kThreads];      // first table entry taken, given
  __shared__ int lens[kThreads];           // positions after
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  long long all[3];  // of a chunk

  // Inclusive sums over a chunk of n sequences, its totals in `all`. A wave's sums fit 32 bits: of entries (each below
  // 2^26), and of token rows (below 2^30) in two halves. (Over the waves that have sequences alone: all 16 for
  // each of three sums took half of a small call's time.)
  auto scan = [&](const Ask& x, int n, long long (&v)[3]) {
    v[0] = wave_scan((uint32_t)x.taken());
    v[1] = wave_scan((uint32_t)x.given());
    v[2] = (long long)wave_scan((uint32_t)x.grown >> 16) * 65536 + wave_scan((uint32_t)x.grown & 0xffff);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (lane == 63) part[k][wv] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) all[k] = 0;
    for (int u = 0; u < (n + kWave - 1) / kWave; ++u) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (u == wv) v[k] += all[k];
        all[k] += part[k][u];
      }
    }
  };

  // ---- the whole batch's totals: does the call go through?
  const long long n_free = max(a.n_free[0], 0);
  long long total[3] = {0, 0, 0};
  bool fits = n_free <= a.capacity;
  Ask x{};
  long long v[3];
  for (int base = 0; base < a.B; base += kThreads) {
    x = ask_of(a, base + tid);
    fits &= __syncthreads_and(x.fits) != 0;
    scan(x, min(a.B - base, kThreads), v);
#pragma unroll
    for (int k = 0; k < 3; ++k) total[k] += all[k];
  }
  const long long top = n_free + total[1], missing = total[0] - top;
  const bool go = fits && missing <= 0 && top <= a.capacity && (a.rows < 0 || total[2] <= a.rows) && total[2] < (1ll << 31);
  if (tid == 0) a.shorts[0] = go ? 0 : missing > 0 ? (int)min(missing, 0x7fffffffll) : -1;
  if (!go) {
    for (int b = tid; b <= a.B; b += kThreads) a.q_start[b] = 0;
    for (int t = tid; with_slots && t < a.rows; t += kThreads) a.slots[t] = -1;
    return;
  }

  // ---- pages given back go to the stack first (from all chunks, as pages taken may be among them), the last sequence's last
  // page lowest: what was taken together comes back as it lay
  int seen[3];
  for (int pass = total[1] > 0 ? 0 : 1; pass < 2; ++pass) {
    seen[0] = seen[1] = seen[2] = 0;
    for (int base = 0; base < a.B; base += kThreads) {
      if (a.B > kThreads) {  // (otherwise the totals' values still stand)
        x = ask_of(a, base + tid);
        __syncthreads();
        scan(x, min(a.B - base, kThreads), v);
      }
      if (a.B > kThreads || pass == 0 || total[1] == 0) {
#pragma unroll
        for (int k = 0; k < 3; ++k) ends[k][tid] = (int)v[k];
        firsts[0][tid] = x.had;
        firsts[1][tid] = x.has;
        lens[tid] = x.len;
        __syncthreads();
      }
      const int n = min(a.B - base, kThreads);
      auto owner = [&](const int* end, int i) {  // the sequence of the chunk whose share holds number i
        int lo = 0, hi = n - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (end[mid] > i)
            hi = mid;
          else
            lo = mid + 1;
        }
        return lo;
      };
      const int k = 1 - pass, moved = ends[k][n - 1];
      int* table = a.table + (size_t)base * a.table_stride;
      int* stack = a.free + (top - 1 - seen[k]);
      for (int i = tid; i < moved; i += kThreads) {
        const int s = owner(ends[k], i);
        int* entry = table + (size_t)s * a.table_stride + (firsts[k][s] + i - (s > 0 ? ends[k][s - 1] : 0));
        if (pass == 0)
          stack[-i] = *entry;
        else
          *entry = stack[-i];
      }
      if (pass == 1) {
        if (tid < n) {
          a.q_start[base + tid + 1] = seen[2] + (int)v[2];
          a.lens[base + tid] = x.len;
        }
        if (with_slots) {
          __syncthreads();  // the entries are written
          const int rows = ends[2][n - 1];
          for (int i = tid; i < rows; i += kThreads) {
            const int s = owner(ends[2], i);
            a.slots[seen[2] + i] = slot_of(a, base + s, lens[s], ends[2][s] - i);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) seen[q] += (int)all[q];
      if (a.B > kThreads) __syncthreads();  // (the arrays are read)
    }
    __syncthreads();
  }
  if (tid == 0) {
    a.q_start[0] = 0;
    a.n_free[0] = (int)(top - total[0]);
  }
  for (long long t = total[2] + tid; with_slots && t < a.rows; t += kThreads) a.slots[t] = -1;
}

// The slot map of long prompts: a thread per token row, behind reserve_kernel.
__global__ void __launch_bounds__(256) slots_kernel(ReserveArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.rows) return;
  long long slot = -1;
  if (t < a.q_start[a.B]) {
    int lo = 0, hi = a.B;  // q_start[lo] <= t < q_start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.q_start[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    slot = slot_of(a, lo, a.lens[lo], a.q_start[lo + 1] - t);
  }
  a.slots[t] = slot;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace ns

extern "C" int ns_paged_reserve(const int* add, int* lens, int* table, long long table_stride, int width,
                                int* free_pages, long long capacity, int* n_free, int* q_start, long long* slots,
                                int rows, int* shorts, int B, int page_size, void* stream) {
  if (B <= 0 || B >= (1 << 24) || width <= 0 || page_size <= 0 || page_size % 16 || capacity < 0 || rows < -1) return -2;
  if ((long long)width * page_size >= (1ll << 30) || table_stride < width || table_stride >> 46 || capacity >= (1ll << 31))
    return -2;
  if (!add || !lens || !table || !n_free || !q_start || !shorts || (!free_pages && capacity > 0)) return -2;
  if (rows > 0 && !slots) return -2;
  for (const void* p : {(const void*)add, (const void*)lens, (const void*)table, (const void*)free_pages,
                        (const void*)n_free, (const void*)q_start, (const void*)shorts})
    if (!ns::aligned(p, 4)) return -2;
  if (!ns::aligned(slots, 8)) return -2;
  const ns::Bytes all[] = {ns::bytes_of(add, 4 * (size_t)B),
                           ns::bytes_of(lens, 4 * (size_t)B),
                           ns::rows_of(table, B, table_stride, width, 4),
                           ns::bytes_of(free_pages, 4 * (size_t)capacity),
                           ns::bytes_of(n_free, 4),
                           ns::bytes_of(q_start, 4 * ((size_t)B + 1)),
                           ns::bytes_of(rows > 0 ? slots : nullptr, 8 * (size_t)std::max(rows, 0)),
                           ns::bytes_of(shorts, 4)};
  for (size_t i = 0; i < std::size(all); ++i)
    for (size_t j = 0; j < i; ++j)
      if (!ns::apart(all[i], all[j])) return -2;
  const ns::ReserveArgs a{add, lens, table, free_pages, n_free, q_start, shorts, slots, table_stride, capacity, B, width,
                          page_size, rows};
  const auto st = static_cast<hipStream_t>(stream);
  const bool own = rows > ns::kOwnRows;
  hipLaunchKernelGGL(ns::reserve_kernel, dim3(1), dim3(ns::kThreads), 0, st, a, rows > 0 && !own);
  if (own) hipLaunchKernelGGL(ns::slots_kernel, dim3((unsigned)((rows + 255ll) / 256)), dim3(256), 0, st, a);
  return static_cast<int>(hipGetLastError());
}
