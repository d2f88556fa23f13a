// Pages of the beams that go on (gfx950; contract in batch_ops.h): table rows of the parents, and copies of the last,
// partly filled page where a beam goes on more than once. The reference keeps one sequence and has no counterpart.
//
// Whole pages are never written again, so beams share them by their tables alone. The last page has to be a beam's own:
// of a parent's children one keeps it, and the others take over the last pages of beams that ended, of which there are as
// many. Sources are thus pages that stay and destinations pages that nobody reads: all copies and tables go in one launch, and
// a second run of the call gives the same. Bound by HBM for many layers (each copied row read once and written once),
// by the latency of parents -> page ids -> rows for few. A wave copies the rows of one layer and head, eight loads in
// flight to a lane and no divisions: with a workgroup per layer and an index per 16 bytes 16 x 8 beams in 28 layers (88 MB)
// took 30.8 us, 16 beams on pages of 16 17.6. Stores pass the caches, which the copies would leave before they are read.
// Measured: 16 x 8 beams 18.3 us, 4.8 TB/s (20.6 with ordinary stores); 4 x 4 beams on pages of 16 4.4 us.
//
// Whole pages that only ended beams had are in no table afterwards. They go to the stack of free pages, where the caller gives
// it: one workgroup looks at every column of the requests' tables, 64 of one request to a wave, and prefix sums say which place
// is whose, so the order is always the same. Bound by the latency of parents -> entries -> others' entries, wave by wave: with
// it 4 beams of 333 positions take 6.5 us instead of 3.3, 16 x 8 beams of 100 to 900 on pages of 64 in 28 layers 23.5 instead of
// 17.6, of 8000 on pages of 16 in one layer 36 instead of 3.2 (52 where half of the columns are each beam's own).
#include <stdint.h>

#include <algorithm>

#include "batch_ops.h"
#include "paged_common.h"

namespace ns {
namespace {

constexpr int kThreads = 256;
constexpr int kMostBeams = 64;

struct ReorderArgs {
  const int *parents, *table, *lens;
  long long parent_stride, table_stride;
  int* out;  // [rows][width]
  uint8_t *pool[2], *scale[2];  // K and V; scales null: a cache without
  long long layer, page, head, s_layer, s_page, s_head;  // strides in bytes
  int beams, width, page_size, row_bytes, n_pages, Hk, layers, groups, table_grid;
};

// Beam i's parent and the beam whose last page it gets, of the request whose lanes hold the parents (lane = beam).
// Every lane of the wave takes part.
struct Way {
  int parent, place;
};
__device__ __forceinline__ Way way_of(const ReorderArgs& a, long long request, int beam) {
  const int lane = __lane_id();
  int p = -1;
  if (lane < a.beams) {
    p = a.parents[request * a.parent_stride + lane];
    if ((unsigned)p >= (unsigned)a.beams) p = lane;  // no parent: goes on as it is
  }
  // the child that keeps the parent's page: the parent itself, or else the first one
  const unsigned long long stays = __ballot(p == lane);
  unsigned long long goes_on = 0, keeps = 0;
  for (int q = 0; q < a.beams; ++q) {
    const unsigned long long children = __ballot(p == q);
    if (!children) continue;
    goes_on |= 1ull << q;
    keeps |= stays >> q & 1 ? 1ull << q : children & -children;
  }
  const unsigned long long all = a.beams == 64 ? ~0ull : (1ull << a.beams) - 1;
  unsigned long long ended = all & ~goes_on, copied = all & ~keeps;
  Way w;
  w.parent = __builtin_amdgcn_readlane(p, beam);
  w.place = w.parent;
  if (copied >> beam & 1) {  // the k-th copy goes to the k-th ended beam's page
    for (int k = __popcll(copied & ((1ull << beam) - 1)); k > 0; --k) ended &= ended - 1;
    w.place = __builtin_ctzll(ended);
  }
  return w;
}

__global__ void __launch_bounds__(kThreads) reorder_kernel(ReorderArgs a) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.table_grid) {  // a workgroup per table row
    const long long row = blockIdx.x, request = row / a.beams;
    const int beam = (int)(row % a.beams);
    const Way w = way_of(a, request, beam);
    const long long from = request * a.beams + w.parent;
    const int len = min(max(a.lens[from], 0), a.width * a.page_size), whole = len / a.page_size;
    for (int j = tid; j < a.width; j += kThreads) {
      const long long src = j < whole ? from : j == whole && len % a.page_size ? request * a.beams + w.place : row;
      a.out[row * a.width + j] = a.table[src * a.table_stride + j];
    }
    return;
  }
  // a wave per beam, layer, head and one of K and V, whose rows are contiguous
  long long id = blockIdx.x - a.table_grid;
  const int kv = (int)(id & 1);
  id >>= 1;
  const int pair = (int)(id % a.groups) * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long row = id / a.groups, request = row / a.beams;
  const Way w = way_of(a, request, (int)(row % a.beams));
  if (w.place == w.parent || pair >= a.layers * a.Hk) return;
  const long long from = request * a.beams + w.parent;
  const int len = min(max(a.lens[from], 0), a.width * a.page_size), part = len % a.page_size;
  if (part == 0) return;
  const int at = len / a.page_size;
  const int src = a.table[from * a.table_stride + at], dst = a.table[(request * a.beams + w.place) * a.table_stride + at];
  if ((unsigned)src >= (unsigned)a.n_pages || (unsigned)dst >= (unsigned)a.n_pages) return;
  const int layer = pair / a.Hk, head = pair % a.Hk, lane = tid & 63;
  uint8_t* rows = a.pool[kv] + layer * a.layer + head * a.head;
  const u32x4_t* s = reinterpret_cast<const u32x4_t*>(rows + src * a.page);
  u32x4_t* d = reinterpret_cast<u32x4_t*>(rows + dst * a.page);
  const int chunks = part * a.row_bytes / 16;  // of 16 bytes
  constexpr int kAtOnce = 8;
  for (int c0 = lane; c0 < chunks; c0 += kAtOnce * kWave) {
    u32x4_t v[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (c0 + u * kWave < chunks) v[u] = s[c0 + u * kWave];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (c0 + u * kWave < chunks) __builtin_nontemporal_store(v[u], &d[c0 + u * kWave]);
  }
  if (!a.scale[kv]) return;
  uint8_t* scales = a.scale[kv] + layer * a.s_layer + head * a.s_head;
  for (int i = lane; i < (part + kScaleRows - 1) / kScaleRows; i += kWave) scales[dst * a.s_page + i] = scales[src * a.s_page + i];
}

constexpr int kBackThreads = 1024, kBackWaves = kBackThreads / kWave;

struct BackArgs {
  const int *parents, *table, *lens;
  long long parent_stride, table_stride, capacity;
  int *free, *n_free;
  int R, beams, width, page_size, n_pages;
};

// The beams, as bits, whose page in column `col` (one to a lane) no beam has that goes on, nor an earlier one of them.
__device__ __forceinline__ unsigned long long dropped_of(const BackArgs& a, long long request, int col) {
  const int lane = __lane_id();
  int p = -1, whole = 0;
  if (lane < a.beams) {
    p = a.parents[request * a.parent_stride + lane];
    if ((unsigned)p >= (unsigned)a.beams) p = lane;
    whole = min(max(a.lens[request * a.beams + lane], 0), a.width * a.page_size) / a.page_size;
  }
  unsigned long long goes_on = 0;
  for (int q = 0; q < a.beams; ++q)
    if (__ballot(p == q)) goes_on |= 1ull << q;
  const unsigned long long all = a.beams == 64 ? ~0ull : (1ull << a.beams) - 1;
  const int* column = a.table + request * a.beams * a.table_stride + min(col, a.width - 1);
  unsigned long long dropped = 0;
  for (unsigned long long ended = all & ~goes_on; ended; ended &= ended - 1) {
    const int e = __builtin_ctzll(ended);
    if (!__any(col < __builtin_amdgcn_readlane(whole, e))) continue;
    const int id = column[e * a.table_stride];
    bool held = col >= __builtin_amdgcn_readlane(whole, e) || (unsigned)id >= (unsigned)a.n_pages;
    // four at a time, the first ones beside the page itself; most columns are shared with one of them
    unsigned long long others = goes_on | (all & ~goes_on & ((1ull << e) - 1));
    do {
      int other[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        other[u] = others ? column[__builtin_ctzll(others) * a.table_stride] : -1;
        others &= others - 1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) held |= other[u] == id;
    } while (others && !__all(held));
    if (!held) dropped |= 1ull << e;
  }
  return dropped;
}

__global__ void __launch_bounds__(kBackThreads) back_kernel(BackArgs a) {
  __shared__ int part[2][kBackWaves];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long chunks = (a.width + kWave - 1) / kWave, tasks = a.R * chunks;
  long long top = max(a.n_free[0], 0);
  if (top > a.capacity) return;
  int now = 0;
  for (long long base = 0; base < tasks; base += kBackWaves, now ^= 1) {
    const long long task = base + wv, request = task / chunks;
    const int col = (int)(task % chunks) * kWave + lane;
    unsigned long long dropped = task < tasks ? dropped_of(a, request, col) : 0;
    const int n = __popcll(dropped), upto = wave_scan(n);
    if (lane == 63) part[now][wv] = upto;
    __syncthreads();  // (the other half is read until here)
    long long at = top + upto - n;
#pragma unroll
    for (int u = 0; u < kBackWaves; ++u) {
      if (u < wv) at += part[now][u];
      top += part[now][u];
    }
    for (; dropped; dropped &= dropped - 1, ++at) {
      const int e = __builtin_ctzll(dropped);
      if (at < a.capacity) a.free[at] = a.table[(request * a.beams + e) * a.table_stride + col];
    }
  }
  __syncthreads();  // (every wave has read the height)
  if (tid == 0) a.n_free[0] = (int)min(top, a.capacity);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Pages, heads and layers of pieces of `piece` bytes: whether no two share a byte, whichever of the dimensions is the
// outer one (each stride spans what the smaller ones span together).
bool nested(long long piece, long long layers, long long layer, long long pages, long long page, long long heads,
            long long head) {
  std::pair<long long, long long> dims[] = {{layer, layers}, {page, pages}, {head, heads}};
  std::sort(std::begin(dims), std::end(dims));
  __int128 span = piece;
  for (const auto& d : dims) {
    if (d.second == 1) continue;
    if (d.first < span) return false;
    span += (__int128)d.first * (d.second - 1);
  }
  return true;
}

// Both entry points; n_free null: no stack.
int reorder(const int* parents, long long parent_stride, const int* table, long long table_stride, int width, const int* lens,
            int* out, void* k_pool, void* v_pool, long long layer_stride, long long page_stride, long long head_stride,
            void* k_scales, void* v_scales, long long scale_layer_stride, long long scale_page_stride,
            long long scale_head_stride, int layers, int n_pages, int page_size, int row_bytes, int R, int beams, int Hk,
            int* free_pages, long long capacity, int* n_free, void* stream) {
  if (R <= 0 || beams <= 0 || beams > kMostBeams || (long long)R * beams >= (1 << 24)) return -2;
  if (width <= 0 || page_size <= 0 || page_size % 16 || (long long)width * page_size >= (1ll << 30)) return -2;
  if (layers <= 0 || n_pages <= 0 || Hk <= 0 || row_bytes <= 0 || row_bytes % 16) return -2;
  if ((long long)page_size * row_bytes * Hk >= (1ll << 31)) return -2;
  if (parent_stride < beams || parent_stride >> 46 || table_stride < width || table_stride >> 46) return -2;
  if (!parents || !table || !lens || !out || !k_pool || !v_pool || !k_scales != !v_scales) return -2;
  for (const void* p : {(const void*)parents, (const void*)table, (const void*)lens, (const void*)out})
    if (!aligned(p, 4)) return -2;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16)) return -2;
  for (const long long s : {layer_stride, page_stride, head_stride})
    if (s < 0 || s % 16 || s >> 46) return -2;
  for (const long long s : {scale_layer_stride, scale_page_stride, scale_head_stride})
    if (s < 0 || s >> 46) return -2;
  const long long piece = (long long)page_size * row_bytes, marks = page_size / kScaleRows, rows = (long long)R * beams;
  if (!nested(piece, layers, layer_stride, n_pages, page_stride, Hk, head_stride)) return -2;
  if (k_scales && !nested(marks, layers, scale_layer_stride, n_pages, scale_page_stride, Hk, scale_head_stride))
    return -2;
  if ((long long)layers * Hk >= (1ll << 30) || rows * (((long long)layers * Hk + 3) / 4 * 2 + 1) >= (1ll << 31)) return -2;
  const Bytes y = bytes_of(out, 4 * (size_t)rows * width), z[] = {rows_of(parents, R, parent_stride, beams, 4),
                                                                        rows_of(table, rows, table_stride, width, 4),
                                                                        bytes_of(lens, 4 * (size_t)rows)};
  for (const Bytes& r : z)
    if (!apart(y, r)) return -2;
  // what lies between the pools' pages counts as theirs here
  auto span = [&](const void* p, long long x, long long layer, long long page, long long head) {
    return bytes_of(p, (layers - 1) * layer + (n_pages - 1) * page + (Hk - 1) * head + x);
  };
  const Bytes pools[] = {span(k_pool, piece, layer_stride, page_stride, head_stride),
                             span(v_pool, piece, layer_stride, page_stride, head_stride),
                             span(k_scales, marks, scale_layer_stride, scale_page_stride, scale_head_stride),
                             span(v_scales, marks, scale_layer_stride, scale_page_stride, scale_head_stride)};
  for (const Bytes& p : pools)
    if (!apart(p, y) || !apart(p, z[0]) || !apart(p, z[1]) || !apart(p, z[2])) return -2;
  if (n_free) {
    if (capacity < 0 || capacity >= (1ll << 31) || (!free_pages && capacity > 0)) return -2;
    if (!aligned(free_pages, 4) || !aligned(n_free, 4)) return -2;
    const Bytes stack[] = {bytes_of(free_pages, 4 * (size_t)capacity), bytes_of(n_free, 4)};
    if (!apart(stack[0], stack[1])) return -2;
    for (const Bytes& r : stack) {
      if (!apart(r, y) || !apart(r, z[0]) || !apart(r, z[1]) || !apart(r, z[2])) return -2;
      for (const Bytes& p : pools)
        if (!apart(r, p)) return -2;
    }
  }
  // but K's, V's and the scales' pages may lie between each other's, if they are equally far apart
  const Pieces codes{{layer_stride, page_stride, head_stride}, {layers, n_pages, Hk}, piece},
      scales{{scale_layer_stride, scale_page_stride, scale_head_stride}, {layers, n_pages, Hk}, marks};
  const bool together = n_pages == 1 || page_stride == scale_page_stride;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (!apart(pools[i], pools[j]) &&
          (((i < 2) != (j < 2) && !together) || !pieces_apart(i < 2 ? codes : scales, j < 2 ? codes : scales,
                                                               (__int128)pools[j].lo - pools[i].lo)))
        return -2;
  ReorderArgs a{};
  a.parents = parents;
  a.table = table;
  a.lens = lens;
  a.parent_stride = parent_stride;
  a.table_stride = table_stride;
  a.out = out;
  a.pool[0] = static_cast<uint8_t*>(k_pool);
  a.pool[1] = static_cast<uint8_t*>(v_pool);
  a.scale[0] = static_cast<uint8_t*>(k_scales);
  a.scale[1] = static_cast<uint8_t*>(v_scales);
  a.layer = layer_stride;
  a.page = page_stride;
  a.head = head_stride;
  a.s_layer = scale_layer_stride;
  a.s_page = scale_page_stride;
  a.s_head = scale_head_stride;
  a.beams = beams;
  a.width = width;
  a.page_size = page_size;
  a.row_bytes = row_bytes;
  a.n_pages = n_pages;
  a.Hk = Hk;
  a.layers = layers;
  a.table_grid = (int)rows;
  a.groups = (int)(((long long)layers * Hk + 3) / 4);
  const auto st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)(rows * (2ll * a.groups + 1))), dim3(kThreads), 0, st, a);
  if (n_free) {
    const BackArgs b{parents, table, lens, parent_stride, table_stride, capacity, free_pages, n_free, R, beams, width, page_size,
                     n_pages};
    hipLaunchKernelGGL(back_kernel, dim3(1), dim3(kBackThreads), 0, st, b);
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace ns

extern "C" {

int ns_paged_reorder(const int* parents, long long parent_stride, const int* table, long long table_stride, int width,
                     const int* lens, int* out, void* k_pool, void* v_pool, long long layer_stride,
                     long long page_stride, long long head_stride, void* k_scales, void* v_scales,
                     long long scale_layer_stride, long long scale_page_stride, long long scale_head_stride, int layers,
                     int n_pages, int page_size, int row_bytes, int R, int beams, int Hk, void* stream) {
  return ns::reorder(parents, parent_stride, table, table_stride, width, lens, out, k_pool, v_pool, layer_stride, page_stride,
                     head_stride, k_scales, v_scales, scale_layer_stride, scale_page_stride, scale_head_stride, layers, n_pages,
                     page_size, row_bytes, R, beams, Hk, nullptr, 0, nullptr, stream);
}

int ns_paged_reorder_back(const int* parents, long long parent_stride, const int* table, long long table_stride, int width,
                          const int* lens, int* out, void* k_pool, void* v_pool, long long layer_stride,
                          long long page_stride, long long head_stride, void* k_scales, void* v_scales,
                          long long scale_layer_stride, long long scale_page_stride, long long scale_head_stride, int layers,
                          int n_pages, int page_size, int row_bytes, int R, int beams, int Hk, int* free_pages,
                          long long capacity, int* n_free, void* stream) {
  if (!n_free) return -2;
  return ns::reorder(parents, parent_stride, table, table_stride, width, lens, out, k_pool, v_pool, layer_stride, page_stride,
                     head_stride, k_scales, v_scales, scale_layer_stride, scale_page_stride, scale_head_stride, layers, n_pages,
                     page_size, row_bytes, R, beams, Hk, free_pages, capacity, n_free, stream);
}

}  // extern "C"
