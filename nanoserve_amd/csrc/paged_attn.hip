// Attention of a batch's new tokens over a paged KV cache (gfx950; contract in batch_ops.h): single
// tokens, prompts, a window with first tokens, and a prefix that all sequences share. The reference
// has PyTorch SDPA over one contiguous cache (python/nanoserve/qwen.py:124-133).
//
// Two launches at most: the keys of the shared prefix (tiles over all tokens' rows) together with each
// sequence's own keys (streamed for single tokens, else tiles), and a merge of the fp32 partials.
//
// Work is dealt out on the device, because lengths are device values (a captured graph replays at any
// lengths): every workgroup adds up the key blocks of the whole batch, takes the share per workgroup
// that spreads them over `target` workgroups, and finds its own sequence, row tile and range of blocks
// by a wave-wide prefix sum over the sequences. One long and fifteen short sequences then end together.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attn_common.h"
#include "batch_ops.h"
#include "paged_common.h"
#include "w4_kernels.h"

namespace ns {
namespace {

constexpr int kTileRows = 128;  // query rows of a tile
constexpr int kTileKeys = 64;   // keys per block of the tile kernel
constexpr int kOneRows = 16;    // cache rows per block of the one-token kernel
constexpr int kOneWaves = 4;
constexpr uint32_t kOut = 0x7fffffffu;  // a buffer offset out of every range: reads as zero

struct PagedArgs {
  const uint16_t* q;
  long long q_stride;
  Batch s;
  Pools p;
  uint16_t* out;
  int4* rows;            // per token row: first partial, their distance, their number
  float *opart, *ml;     // own keys: [cap][Hq][D] and [cap][Hq][2] (maximum, sum)
  float *shpart, *shml;  // shared keys: [splits][T][Hq][D] and [..][2]
  long long cap;
  int Hq, Hk, R, shared, window, sinks, sh_splits, sh_grid, unit;
  float per_target;  // kv heads / workgroups aimed at
  float c;           // scale * log2(e)
};

// LDS of a workgroup: 64 KiB (D = 128: two stages of 64 rows of K and of V; D = 64: four). Separate arrays,
// not one: where a read of a stage provably does not alias the loads in flight into another, the compiler puts
// no wait for those before it. It still puts some, which hold the ring below its depth: in the one-token kernel
// before the reads of stage 0 (vmcnt 1 before K, 0 before V; with two stages the other's loads are then drained in every
// second block), and in tiles of four stages in every block, behind the loads just sent out (vmcnt 3 to 0 before
// the scores: the query fragments, loaded before the ring, may for all it knows be in flight behind the ring's
// conditional waits). Tiles of two stages, whose wait is for all loads, have none.
template <int D>
constexpr int ring_stages() {
  return D == 128 ? 2 : 4;
}
struct Ring {
  uint16_t *k[4], *v[4];
};
// Of a tile over the shared prefix: each row's positions (from, up to; the first tokens besides), and the least
// and highest of each wave's.
struct SharedRows {
  int2 limits[kTileRows];
  int lim[4][2];
};

// The key blocks that some query of a range sees: positions k0 .. k1 - 1, of them those below `first`
// or from `lo` on.
template <int BLK>
struct KeyBlocks {
  int a0, na, m0, nm;
  __device__ KeyBlocks(int k0, int k1, int lo, int first) {
    a0 = k0 / BLK;
    const int e0 = min(min(first, lo), k1) > k0 ? (min(min(first, lo), k1) + BLK - 1) / BLK : a0;
    m0 = max(max(lo, k0) / BLK, e0);
    na = k1 > k0 ? e0 - a0 : 0;
    nm = k1 > k0 ? max((k1 + BLK - 1) / BLK - m0, 0) : 0;
  }
  __device__ int count() const { return na + nm; }
  __device__ int block(int j) const { return j < na ? a0 + j : m0 + j - na; }
};

// The largest of the lanes' values, none below 0 (lanes shifted in from outside count as 0).
__device__ __forceinline__ int wave_most(int m) {
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x111, 0xf, 0xf, false));
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x112, 0xf, 0xf, false));
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x114, 0xf, 0xf, false));
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x118, 0xf, 0xf, false));
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x142, 0xa, 0xf, false));
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(m, 63);
}

// One of the longest sequences: its table row has every shared position that any sequence has.
__device__ __forceinline__ int longest(const PagedArgs& a) {
  const int lane = __lane_id();
  int most = -1, at = 0;
  for (int b = lane; b < a.s.B; b += kWave) {
    const int n = a.s.positions(b);
    if (n > most) {
      most = n;
      at = b;
    }
  }
  return __builtin_amdgcn_readlane(at, __builtin_ctzll(__ballot(most == wave_most(max(most, 0)))));
}

__device__ __forceinline__ int low_limit(const PagedArgs& a, int pos) {
  return a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
}

// One sequence's share of the launch. ROWS 0: one token per sequence and all its rows in one tile.
struct Span {
  int n, row0, nn, tiles, blocks, splits;
};

template <int BLK, int ROWS>
__device__ __forceinline__ Span span_of(const PagedArgs& a, int b) {
  Span x;
  x.n = a.s.positions(b);
  a.s.tokens(b, x.row0, x.nn);
  x.tiles = ROWS ? (x.nn * a.R + max(ROWS, 1) - 1) / max(ROWS, 1) : x.nn;
  // blocks of the last tile, the longest one; the other tiles' lists are split into as many ranges
  const int toks = ROWS ? min(x.nn, max(ROWS, 1) / a.R + 1) : 1;
  x.blocks = KeyBlocks<BLK>(a.shared, x.n, low_limit(a, x.n - toks), a.window > 0 ? a.sinks : 0).count();
  x.splits = 0;
  return x;
}

// Inclusive prefix sums over the wave by DPP (row shifts, then row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Item `item` of the batch: its sequence, the number within it, and the sequence's first partial (a
// token slot). False past the last item. Uniform over the workgroup's waves.
template <int BLK, int ROWS>
__device__ __forceinline__ bool find_item(const PagedArgs& a, int item, int& b, Span& sp, int& within,
                                          long long& slot) {
  const int lane = __lane_id(), B = a.s.B;
  Span x{};
  float total = 0.f, tiles = 0.f;  // (every wave of the launch adds the same values in the same order)
  for (int base = 0; base < B; base += kWave) {
    x = Span{};
    if (base + lane < B) x = span_of<BLK, ROWS>(a, base + lane);
    total += (float)x.tiles * (float)x.blocks;
    tiles += (float)x.tiles;
  }
  total = wave_sum(total);
  const int share = __builtin_amdgcn_readfirstlane((int)ceilf(total * a.per_target));
  int per = max(a.unit, (share + a.unit - 1) / a.unit * a.unit);
  // Sequences end inside a share: where that makes more items than workgroups aimed at, the last ones would
  // start when the others end. Larger shares then, a few times at most, if the items can be that few at all
  // (us without and with: 64 sequences of 1000 to 8000 positions 118.7, 110.0; 20 of 1000 to 4000 with 8 kv
  // heads 41.9, 38.5; 200 of up to 1000, whose 800 items are more anyway, 51.6, 59.0).
  const bool fits = B <= 4 * kWave && wave_sum(tiles) * a.per_target < 0.9f;
#pragma unroll 1
  for (int step = 0; step < 3 && fits; ++step) {
    int items = 0;
    for (int base = 0; base < B; base += kWave) {
      if (B > kWave) {
        x = Span{};
        if (base + lane < B) x = span_of<BLK, ROWS>(a, base + lane);
      }
      items += x.nn > 0 ? x.tiles * max(1, (x.blocks + per - 1) / per) : 0;
    }
    const float over = (float)__builtin_amdgcn_readlane(wave_scan(items), kWave - 1) * a.per_target;
    if (over <= 1.f) break;
    per = ((int)((float)per * fminf(over, 2.f)) / a.unit + 1) * a.unit;
  }

  int seen = 0;
  slot = 0;
  for (int base = 0; base < B; base += kWave) {
    if (B > kWave) {
      x = Span{};
      if (base + lane < B) x = span_of<BLK, ROWS>(a, base + lane);
    }
    x.splits = x.nn > 0 ? max(1, (x.blocks + per - 1) / per) : 0;
    const int items = x.tiles * x.splits, slots = x.nn * x.splits;
    const int upto = wave_scan(items), all = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (item < seen + all) {
      const int src = __builtin_ctzll(__ballot(seen + upto > item));
      b = base + src;
      within = item - seen - __builtin_amdgcn_readlane(upto - items, src);
      sp.n = __builtin_amdgcn_readlane(x.n, src);
      sp.row0 = __builtin_amdgcn_readlane(x.row0, src);
      sp.nn = __builtin_amdgcn_readlane(x.nn, src);
      sp.tiles = __builtin_amdgcn_readlane(x.tiles, src);
      sp.blocks = __builtin_amdgcn_readlane(x.blocks, src);
      sp.splits = __builtin_amdgcn_readlane(x.splits, src);
      slot += __builtin_amdgcn_readlane(wave_scan(slots) - slots, src);
      return true;
    }
    seen += all;
    slot += __builtin_amdgcn_readlane(wave_scan(slots), kWave - 1);
  }
  return false;
}

// The lanes' bits together.
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
  v |= __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v |= __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v |= __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v |= __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v |= __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v |= __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return __builtin_amdgcn_readlane(v, 63);
}

// attn_lds_load16 for rows that one workgroup reads, once.
__device__ __forceinline__ void lds_stream16(__amdgpu_buffer_rsrc_t r, uint16_t* dst, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0,
                                           kStreamAux);
}

// A block's loads have landed when at most n newer ones of this wave are in flight (n a multiple of 4
// below 16).
__device__ __forceinline__ void wait_loads(int n) {
  if (n >= 12)
    __builtin_amdgcn_s_waitcnt(0x0F7C);
  else if (n >= 8)
    __builtin_amdgcn_s_waitcnt(0x0F78);
  else if (n >= 4)
    __builtin_amdgcn_s_waitcnt(0x0F74);
  else
    __builtin_amdgcn_s_waitcnt(0x0F70);
  asm volatile("" ::: "memory");
}

// The maximum that stands for a range of keys from here on: -inf if and only if the row sees none of them. Scores
// that are all -inf, or all NaN (which fmaxf passes over), leave -inf too; the lowest finite value in its place
// keeps their sums (0 and NaN) in the merge, where they weigh nothing beside finite scores (0 * NaN is NaN) and
// divide 0 by 0 alone.
__device__ __forceinline__ float seen_max(float m, bool seen) { return seen ? fmaxf(m, -FLT_MAX) : -INFINITY; }

// ------------------------------------------------------------------ one token per sequence
// Up to 16 query heads per kv head, bound by HBM. A workgroup takes a range of 16-row blocks of one
// sequence and kv head; each of its four waves streams every fourth block through its own LDS ring
// (K and V by buffer-to-LDS loads, waiting only for its own; 64 KiB per workgroup at D = 128, two
// workgroups per CU). A block lies in one page, whose id is a scalar: lanes hold the wave's next 64 ids.
//  * Scores: K rows as the A operand, the heads as columns (v_mfma_f32_16x16x32_bf16); a lane then has
//    four keys of one head. Values: probabilities as the A operand of v_mfma_f32_16x16x16_bf16, V by
//    transposed LDS reads. Probabilities enter as two bf16 terms (p to within 2^-16 of it), so that the
//    product is as exact as the fp32 softmax before it; the matrix cores idle at HBM's pace anyway.
//  * LDS rows are D / 8 chunks of 16 B, XOR-swizzled: K rows by their number (the 16 rows of a fragment
//    read hit distinct banks), V rows so that the 4 x 16 blocks of a transposed read do.
//  * Value rows that the token does not see are not read but zero: their probability is 0, and whatever
//    the page holds there (it may be NaN) must not reach the sum.
// Measured (28 / 4 heads of 128): 4 sequences of 98 000 127 us, 6.2 TB/s of reads (a read probe reaches 6.84); 32
// of 3000 to 30000 with a window of 4096 52.6 us, 5.1 TB/s; 16 of 33 to 8191 30 us, of them 4 in the merge; one of
// 700 with 12 / 2 heads 9.4 us, the latency of two launches.
template <int D>
__device__ __forceinline__ void one_body(const PagedArgs& a, int item, int g, const Ring& lds,
                                         float (&red)[2][kOneWaves][16]) {
  constexpr int kBlk = kOneRows * D, kChunks = D / 8, kRowsPerLoad = 64 / kChunks,
                kLoads = kOneRows / kRowsPerLoad, kStages = ring_stages<D>();
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.R;
  int b, split;
  long long slot;
  Span sp;
  if (!find_item<kOneRows, 0>(a, item, b, sp, split, slot)) return;
  const bool direct = sp.splits == 1 && a.sh_splits == 0;
  if (!direct && (slot < 0 || slot + sp.splits > a.cap)) return;

  const int n = sp.n, lo = low_limit(a, n - 1), first = a.window > 0 ? a.sinks : 0, k0 = a.shared;
  const KeyBlocks<kOneRows> kb(k0, n, lo, first);
  const int j0 = (int)((long long)kb.count() * split / sp.splits);
  const int j1 = (int)((long long)kb.count() * (split + 1) / sp.splits);
  const int cnt = j1 - j0 > wv ? (j1 - j0 - wv + kOneWaves - 1) / kOneWaves : 0;  // this wave's blocks

  // B operand of the scores: lane (head l % 16, grp = l / 16), dims 32 s + 8 grp ..; heads past R: 0
  const int r16 = lane & 15, grp = lane >> 4;
  u32x4_t qf[D / 32];
  {
    const uint16_t* qp = a.q + (size_t)b * a.q_stride + (size_t)(g * R + min(r16, R - 1)) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(qp + 32 * s);
      qf[s] = r16 < R ? v : u32x4_t{0u, 0u, 0u, 0u};
    }
  }

  // lane i: offset in the pools and first position of the wave's block 64 (.. / 64) + i; no page: position -1
  const int* table = a.s.table + (size_t)b * a.s.table_stride;
  uint64_t offs = 0;
  int keys = -1;
  auto refill = [&](int i) {
    const int v = i + lane;
    if (v < cnt) {
      keys = kOneRows * kb.block(j0 + wv + kOneWaves * v);
      const int id = table[keys / a.s.page_size];
      offs = 2 * ((uint64_t)(uint32_t)id * a.p.page_stride + (uint64_t)g * a.p.head_stride +
                  (uint64_t)(keys % a.s.page_size) * D);
      if ((unsigned)id >= (unsigned)a.p.n_pages) keys = -1;
    }
  };
  auto k_swz = [](int row) { return D == 128 ? row & 15 : (row >> 1) & 7; };
  auto v_swz = [](int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); };
  auto seen_key = [&](int key) { return (key < n) & (key >= k0) & ((key >= lo) | (key < first)); };
  auto whole = [&](int key0) { return key0 >= k0 && key0 >= lo && key0 + kOneRows <= n; };
  uint32_t k_off[kLoads], v_off[kLoads];  // of this lane's 16 bytes in a block
  const int lr = lane / kChunks;
#pragma unroll
  for (int p = 0; p < kLoads; ++p) {
    const int row = kRowsPerLoad * p + lr;
    const uint32_t ch = lane % kChunks;
    k_off[p] = row * 2 * D + 16u * (ch ^ k_swz(row));
    v_off[p] = row * 2 * D + 16u * (ch ^ v_swz(row));
  }
  auto issue = [&](uint16_t* ks, uint16_t* vs, int i) {
    if ((i & 63) == 0) refill(i);
    const int key0 = __builtin_amdgcn_readlane(keys, i & 63);
    const bool ok = key0 >= 0;
    const uint64_t off = ok ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(offs >> 32), i & 63) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((uint32_t)offs, i & 63)
                            : 0;
    const auto kres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.k) + off, (short)0,
                                                        ok ? kBlk * 2 : 0, 0x00020000);
    const auto vres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.v) + off, (short)0,
                                                        ok ? kBlk * 2 : 0, 0x00020000);
#pragma unroll
    for (int p = 0; p < kLoads; ++p) lds_stream16(kres, ks + 512 * p, k_off[p]);
    if (whole(key0)) {
#pragma unroll
      for (int p = 0; p < kLoads; ++p) lds_stream16(vres, vs + 512 * p, v_off[p]);
    } else {
#pragma unroll
      for (int p = 0; p < kLoads; ++p)
        lds_stream16(vres, vs + 512 * p, seen_key(key0 + kRowsPerLoad * p + lr) ? v_off[p] : kOut);
    }
  };

  f32x4_t o[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // of head r16
  bool seen = false;             // a block of the wave had a page, and so a key that the token sees
  const int vrow = 4 * grp + (r16 >> 2);
  auto compute = [&](const uint16_t* ks, const uint16_t* vs, int key0) {
    f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(ks + r16 * D + 8 * ((4 * s + grp) ^ k_swz(r16)));
      sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf),
                                                   __builtin_bit_cast(bf16x8_t, qf[s]), sc, 0, 0, 0);
    }
    float sr[4], bm = -INFINITY;  // head r16, keys 4 grp + r (base-2 logits)
#pragma unroll
    for (int r = 0; r < 4; ++r) sr[r] = sc[r] * a.c;
    if (!whole(key0)) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sr[r] = (key0 >= 0) & seen_key(key0 + 4 * grp + r) ? sr[r] : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) bm = fmaxf(bm, sr[r]);
    bm = fmaxf(bm, lane_xor16(bm));
    bm = fmaxf(bm, lane_xor32(bm));
    const float mn = fmaxf(m, bm);
    if (__any(mn > m)) {
      // o holds heads 4 grp + r of dim r16: their factors come from lanes 4 grp + r
      const float alpha = exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = __shfl(alpha, 4 * grp + r, kWave);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[d][r] *= f;
      }
    }
    const float mz = m == -INFINITY ? 0.f : m;
    float ph[4], pl[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float p = exp2f(sr[r] - mz);
      l += p;  // this lane's keys; the lanes are added at the end
      ph[r] = round_bf16(p);
      pl[r] = p - ph[r];
    }
    const s16x4_t pah = __builtin_bit_cast(
        s16x4_t, make_uint2(pack_bf16x2_rne(ph[0], ph[1]), pack_bf16x2_rne(ph[2], ph[3])));
    const s16x4_t pal = __builtin_bit_cast(
        s16x4_t, make_uint2(pack_bf16x2_rne(pl[0], pl[1]), pack_bf16x2_rne(pl[2], pl[3])));
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int chunk = (2 * d + ((lane & 3) >> 1)) ^ v_swz(vrow);
      const s16x4_t vb = __builtin_bit_cast(
          s16x4_t, lds_read_tr16(vs + vrow * D + 8 * chunk + 4 * (lane & 1)));
      o[d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(pah, vb, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(pal, vb, o[d], 0, 0, 0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is read before it is loaded again
    asm volatile("" ::: "memory");
  };

  int at[kStages];  // first positions of the blocks in flight
  auto start = [&](auto stage, int i) {
    constexpr int S = decltype(stage)::value;
    issue(lds.k[S] + wv * kBlk, lds.v[S] + wv * kBlk, i);
    at[S] = __builtin_amdgcn_readlane(keys, i & 63);
  };
  auto step = [&](auto stage, int i) {
    constexpr int S = decltype(stage)::value;
    wait_loads(2 * kLoads * min(cnt - 1 - i, kStages - 1));
    seen |= at[S] >= 0;
    compute(lds.k[S] + wv * kBlk, lds.v[S] + wv * kBlk, at[S]);
    if (i + kStages < cnt) start(stage, i + kStages);
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, (kStages > 2 ? 2 : 0)>;
  using S3 = std::integral_constant<int, (kStages > 2 ? 3 : 0)>;
  if (cnt > 0) start(S0{}, 0);
  if (cnt > 1) start(S1{}, 1);
  if constexpr (kStages > 2) {
    if (cnt > 2) start(S2{}, 2);
    if (cnt > 3) start(S3{}, 3);
  }
  for (int i = 0; i < cnt; i += kStages) {
    step(S0{}, i);
    if (i + 1 < cnt) step(S1{}, i + 1);
    if constexpr (kStages > 2) {
      if (i + 2 < cnt) step(S2{}, i + 2);
      if (i + 3 < cnt) step(S3{}, i + 3);
    }
  }
  l += lane_xor16(l);
  l += lane_xor32(l);
  m = seen_max(m, seen);

  // ---- merge of the waves through their (then free) first stages: fp32, heads 0 .. 7 in the K half and
  // 8 .. 15 in the V half
  auto (&red_m) = red[0];
  auto (&red_l) = red[1];
  float *ok = reinterpret_cast<float*>(lds.k[0]), *ov_ = reinterpret_cast<float*>(lds.v[0]);
  float* half = (grp < 2 ? ok : ov_) + wv * kBlk / 2 + (4 * grp & 7) * D;
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) half[r * D + 16 * d + r16] = o[d][r];
  if (grp == 0) {
    red_m[wv][r16] = m;
    red_l[wv][r16] = l;
  }
  lds_sync();
  for (int i = tid; i < R * D; i += kOneWaves * kWave) {
    const int hh = i / D, d = i % D;
    float mt = red_m[0][hh];
#pragma unroll
    for (int k = 1; k < kOneWaves; ++k) mt = fmaxf(mt, red_m[k][hh]);
    const float mz = mt == -INFINITY ? 0.f : mt;
    float ov = 0.f, lt = 0.f;
#pragma unroll
    for (int k = 0; k < kOneWaves; ++k) {
      const float f = exp2f(red_m[k][hh] - mz);  // 0 for a wave without keys
      ov = fmaf(f, (hh < 8 ? ok : ov_)[k * kBlk / 2 + (hh & 7) * D + d], ov);
      lt = fmaf(f, red_l[k][hh], lt);
    }
    const int h = g * R + hh;
    if (direct) {
      a.out[((size_t)b * a.Hq + h) * D + d] =
          static_cast<uint16_t>(f32_to_bf16_rne(mt == -INFINITY ? 0.f : ov / lt));
    } else {
      const size_t row = (size_t)(slot + split) * a.Hq + h;
      a.opart[row * D + d] = ov;
      if (d == 0) *reinterpret_cast<float2*>(&a.ml[row * 2]) = make_float2(mt, lt);
    }
  }
  // (also where the result is final, so that the merge does not read an older launch's entry)
  if (a.rows && split == 0 && g == 0 && tid == 0) a.rows[b] = make_int4((int)slot, 1, sp.splits, 0);
}

// ------------------------------------------------------------------ tiles of query rows
// Bound by the matrix cores and the softmax's VALU work beside them. The rows of a kv head's problem are its R query heads'
// tokens, token-major (row = token * R + head): one K / V tile serves all heads of the group. kShared:
// the rows of all tokens of the batch over the shared prefix's keys; else one sequence's tokens over
// its own keys.
//  * Workgroup: 128 rows (four waves of 32) over a range of 64-key blocks, two LDS stages (64 KiB at
//    D = 128, two workgroups per CU). A wave loads 16 rows of K and of V per block, which lie in one
//    page; lanes hold the next 16 blocks' page ids.
//  * Scores are computed transposed, S^T = K Q^T on v_mfma_f32_32x32x16_bf16: a lane owns one query and
//    16 of each 32 keys, so the softmax needs one lane swap per reduction and the score registers are,
//    as they stand, the B operand of O^T = V^T P^T; ds_read_b64_tr_b16 delivers V^T's fragments.
//  * Probabilities enter as two bf16 terms (16 significant bits): the error is then the output's own rounding, for
//    1.5 times the products of one term.
//  * A row sees positions below `hi` and from `lo` on or below `sinks`; blocks that no row of the tile
//    sees are left out of its list, blocks that all rows see whole skip the comparisons. Windows of different
//    sequences over the shared prefix may lie apart: the positions between them stay in the list, and their rows
//    are not read but zero, as a value there (it may be NaN) would reach every row through 0 * NaN.
// Measured (28 / 4 heads of 128): prompts of 5 sequences of 2000 to 8000 654 us, 677 TFLOP/s, with the second term
// 1015 (a large library product: 1265); matrix cores busy in half of the cycles and vector units in 58 %, at 1.8 GHz,
// so that products and softmax still take turns for much of the time. Issuing one half block's softmax between the
// products of its neighbours did not help (659 -> 681 to 730 us). 4095 tokens with a window of 1000 and 14 / 2 heads of
// 64 43 us. 96 drafts of 1 to 3 tokens behind 16384 shared positions 100 to 104 us back to back, 108 to 117 among
// other launches: 220 workgroups of the shared keys, one to a CU, with one wave per SIMD.
template <int D, bool kShared>
__device__ __forceinline__ void tile_body(const PagedArgs& a, int item, int g, const Ring& lds, SharedRows& sh) {
  constexpr int kChunks = D / 8, kRowsPerLoad = 64 / kChunks, kLoads = 16 / kRowsPerLoad, kDT = D / 32,
                kStages = ring_stages<D>();
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.R;
  const int jq = lane & 31, kh = lane >> 5;

  int split, splits, r0, rows, k0, k1;
  long long slot = 0;
  Span sp{};
  int b = 0;
  if constexpr (kShared) {
    const int tiles = (a.s.T * R + kTileRows - 1) / kTileRows;
    split = item / tiles;
    splits = a.sh_splits;
    r0 = item % tiles * kTileRows;
    rows = a.s.T * R;
    k0 = 0;
    k1 = min(a.shared, a.s.width * a.s.page_size);
    b = longest(a);
  } else {
    int within;
    if (!find_item<kTileKeys, kTileRows>(a, item, b, sp, within, slot)) return;
    splits = sp.splits;
    split = within % splits;
    r0 = (sp.tiles - 1 - within / splits) * kTileRows;  // longest tiles first
    rows = sp.nn * R;
    k0 = a.shared;
    k1 = sp.n;
  }
  const bool direct = !kShared && splits == 1 && a.sh_splits == 0;
  if (!kShared && !direct && (slot < 0 || slot + (long long)sp.nn * splits > a.cap)) return;

  // this lane's query: rows past the end repeat the last and see nothing
  const int wrow = r0 + 32 * wv;
  const int row = min(wrow + jq, rows - 1);
  const int tok = row / R, hq = g * R + row % R;
  int t, pos;
  bool counts = wrow + jq < rows;  // a row with a result, which is zero if it sees nothing
  if constexpr (kShared) {
    t = tok;
    const int sb = a.s.sequence(t);
    pos = -1;
    counts &= sb >= 0;
    if (sb >= 0) {
      int row0, nn;
      a.s.tokens(sb, row0, nn);
      pos = a.s.positions(sb) - nn + t - row0;
    }
  } else {
    t = sp.row0 + tok;
    pos = sp.n - sp.nn + tok;
  }
  const bool real = counts && pos >= 0;
  const int hi = real ? min(pos + 1, k1) : 0, lo = low_limit(a, pos);
  const int first = a.window > 0 ? a.sinks : 0;
  // limits over the wave's rows and over the tile's: a sequence's positions rise with its rows, the rows of
  // the whole batch need a look at each
  int hi_min, hi_max, lo_min, lo_max, top, low;
  bool gaps = false;  // there may be positions between the rows' windows that no row sees
  if constexpr (kShared) {
    // (a row whose window begins past the prefix sees the first tokens of it alone)
    const int far = a.s.width * a.s.page_size;
    hi_min = k1 - wave_most(counts ? k1 - hi : 0);
    hi_max = wave_most(lo < hi ? hi : min(first, hi));
    lo_min = far - wave_most(real ? far - lo : 0);
    lo_max = wave_most(real ? lo : 0);
    if (kh == 0) sh.limits[32 * wv + jq] = make_int2(lo, hi);
    if (lane == 0) {
      sh.lim[wv][0] = hi_max;
      sh.lim[wv][1] = lo_min;
    }
    lds_sync();
    top = __builtin_amdgcn_readfirstlane(max(max(sh.lim[0][0], sh.lim[1][0]), max(sh.lim[2][0], sh.lim[3][0])));
    if (a.window > 0) {  // none if every window begins at or before the first end of one
      int start = 0, back = 0;
#pragma unroll
      for (int u = 0; u < kTileRows; u += kWave) {
        const int2 x = sh.limits[u + lane];
        start = max(start, x.x < x.y ? x.x : 0);
        back = max(back, x.x < x.y ? k1 - x.y : 0);
      }
      gaps = wave_most(start) + wave_most(back) > k1;
    }
    low = __builtin_amdgcn_readfirstlane(min(min(sh.lim[0][1], sh.lim[1][1]), min(sh.lim[2][1], sh.lim[3][1])));
  } else {
    const int p0 = sp.n - sp.nn;  // of the sequence's first new token; below 0 with more of them than positions
    const int wfirst = p0 + min(wrow, rows - 1) / R, wlast = p0 + min(wrow + 31, rows - 1) / R;
    hi_min = wrow + 31 < rows && wfirst >= 0 ? wfirst + 1 : 0;  // (0: some lane's row sees nothing)
    hi_max = wrow < rows ? max(wlast + 1, 0) : 0;
    lo_min = low_limit(a, wfirst);
    lo_max = low_limit(a, wlast);
    top = max(p0 + min(r0 + kTileRows - 1, rows - 1) / R + 1, 0);
    low = low_limit(a, p0 + r0 / R);
  }
  const KeyBlocks<kTileKeys> kb(k0, top, low, first);
  const int j0 = (int)((long long)kb.count() * split / splits);
  const int j1 = (int)((long long)kb.count() * (split + 1) / splits);

  // B operand of the scores: this lane's query at dims 16 s + 8 kh ..
  u32x4_t qf[D / 16];
  {
    const uint16_t* qp = a.q + (size_t)t * a.q_stride + (size_t)hq * D + 8 * kh;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(qp + 16 * s);
  }

  // lane i: offset in the pools of 16-row group i % 4 of block j0 + 16 (.. / 16) + i / 4 of the list
  const int* table = a.s.table + (size_t)b * a.s.table_stride;
  uint64_t offs = 0, valid = 0;
  auto refill = [&](int j) {
    const int v = j + (lane >> 2);
    int id = -1;
    if (v < j1) {
      const int key = kTileKeys * kb.block(v) + 16 * (lane & 3);
      if (key < top) id = table[key / a.s.page_size];
      offs = 2 * ((uint64_t)(uint32_t)id * a.p.page_stride + (uint64_t)g * a.p.head_stride +
                  (uint64_t)(key % a.s.page_size) * D);
    }
    valid = __ballot((unsigned)id < (unsigned)a.p.n_pages);
  };
  auto k_swz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  auto v_swz = [](int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; };
  uint32_t k_off[kLoads], v_off[kLoads];  // of this lane's 16 bytes in a group
  const int lr = lane / kChunks;
#pragma unroll
  for (int p = 0; p < kLoads; ++p) {
    const int r = kRowsPerLoad * p + lr;
    const uint32_t ch = lane % kChunks;
    k_off[p] = r * 2 * D + 16u * (ch ^ k_swz(16 * wv + r));
    v_off[p] = r * 2 * D + 16u * (ch ^ v_swz(r));
  }
  // Bit i: some row of the tile sees position key0 + i, i < 16.
  auto seen16 = [&](int key0) {
    auto below = [&](int limit) { return (1u << min(max(limit - key0, 0), 16)) - 1; };
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kTileRows; u += kWave) {
      const int2 x = sh.limits[u + lane];
      bits |= (below(x.y) & ~below(x.x)) | below(min(first, x.y));
    }
    return wave_or(bits);
  };
  auto issue = [&](uint16_t* ks, uint16_t* vs, int j, uint32_t& groups) {
    const int jj = j - j0;
    if ((jj & 15) == 0) refill(j);
    const int e = 4 * (jj & 15);
    groups = (uint32_t)(valid >> e) & 15u;
    const int key0 = kTileKeys * kb.block(j) + 16 * wv;
    uint32_t sees = 0xffffu;
    if constexpr (kShared)
      if (gaps) sees = seen16(key0);
    const bool ok = ((groups >> wv) & 1) != 0 && sees != 0;
    const uint64_t off = ok ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(offs >> 32), e + wv) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((uint32_t)offs, e + wv)
                            : 0;
    const auto kres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.k) + off, (short)0,
                                                        ok ? 32 * D : 0, 0x00020000);
    const auto vres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.v) + off, (short)0,
                                                        ok ? 32 * D : 0, 0x00020000);
#pragma unroll
    for (int p = 0; p < kLoads; ++p) attn_lds_load16(kres, &ks[16 * wv * D + 512 * p], k_off[p], 0);
    if (gaps ? sees == 0xffffu : key0 >= k0 && key0 >= low && key0 + 16 <= top) {
#pragma unroll
      for (int p = 0; p < kLoads; ++p) attn_lds_load16(vres, &vs[16 * wv * D + 512 * p], v_off[p], 0);
    } else {  // value rows that no row of the tile sees are zero, whatever the page holds
#pragma unroll
      for (int p = 0; p < kLoads; ++p) {
        const int key = key0 + kRowsPerLoad * p + lr;
        const bool see = gaps ? ((sees >> (key - key0)) & 1) != 0
                              : (key >= k0) & (key < top) & ((key >= low) | (key < first));
        attn_lds_load16(vres, &vs[16 * wv * D + 512 * p], see ? v_off[p] : kOut, 0);
      }
    }
  };

  f32x16_t o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = a.c;

  // transpose-read offsets (elements) of the 32-dim tiles at key row 4 kh + (lane % 16) / 4
  int vt[kDT];
  {
    const int rr = 4 * kh + ((lane & 15) >> 2);
#pragma unroll
    for (int d = 0; d < kDT; ++d)
      vt[d] = rr * D + 8 * ((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swz(rr)) + 4 * (lane & 1);
  }

  auto compute = [&](const uint16_t* kt, const uint16_t* vb, int j, uint32_t groups) {
    const int key0 = kTileKeys * kb.block(j);
    if (key0 >= hi_max || (key0 + kTileKeys <= lo_min && key0 >= first)) return;  // no row sees it
    f32x16_t s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const int kr = 32 * u + jq;
        const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(&kt[kr * D + 8 * ((2 * d + kh) ^ k_swz(kr))]);
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf),
                                                       __builtin_bit_cast(bf16x8_t, qf[d]), s[u], 0, 0, 0);
      }
    }
    // (flags from bitwise operators and one comparison: with && this compiler builds a branch per value, and
    // some of those lost their store)
    if (groups != 15u || (key0 < first && lo_max > 0)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = key0 + 32 * u + 8 * (r >> 2) + 4 * kh + (r & 3);
          const bool see = (key < hi) & (key >= k0) & ((key >= lo) | (key < first)) &
                           (((groups >> (2 * u + (r >> 3))) & 1) != 0);
          s[u][r] = see ? s[u][r] : -INFINITY;
        }
    } else if (key0 + kTileKeys > hi_min || key0 < lo_max || key0 < k0) {  // positions from, .. to - 1
      const int from = max(lo, k0);
      const uint32_t span = (uint32_t)max(hi - from, 0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t at = (uint32_t)(key0 + 4 * kh - from + 32 * u + 8 * (r >> 2) + (r & 3));
          s[u][r] = at < span ? s[u][r] : -INFINITY;
        }
    }
    float bm = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) bm = fmaxf(bm, s[u][r]);
    bm = fmaxf(bm, lane_xor32(bm));
    if (__any(bm > m)) {
      const float mn = fmaxf(m, bm);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f((m - ms) * c);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    u32x4_t pt[2][4];  // B operands of the four 16-key steps
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[u][r + 1], c, -mc));
        l += p0 + p1;
        const uint32_t term = pack_bf16x2_rne(p0, p1);
        pt[0][2 * u + (r >> 3)][(r & 7) >> 1] = term;
        pt[1][2 * u + (r >> 3)][(r & 7) >> 1] = pack_bf16x2_rne(p0 - __uint_as_float(term << 16),
                                                                p1 - __uint_as_float(term & 0xffff0000u));
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8_t vf[kDT];
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        const u32x2_t v0 = lds_read_tr16(&vb[vt[d] + 16 * u * D]);
        const u32x2_t v1 = lds_read_tr16(&vb[vt[d] + (16 * u + 8) * D]);
        vf[d] = __builtin_bit_cast(bf16x8_t, (u32x4_t){v0[0], v0[1], v1[0], v1[1]});
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < kDT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[d], __builtin_bit_cast(bf16x8_t, pt[i][u]), o[d], 0, 0, 0);
    }
  };

  // Block j is ready once every wave's loads of it have landed (those of up to kStages - 2 newer blocks stay
  // in flight), and past the barrier nobody reads block j - 1, whose stage is loaded next: each wave waits for
  // its loads of j and its reads of j - 1.
  uint32_t gr[kStages];
  auto fill = [&](auto stage, int j) {
    constexpr int S = decltype(stage)::value;
    if (j < j1) issue(lds.k[S], lds.v[S], j, gr[S]);
  };
  auto step = [&](auto stage, auto last, int j) {
    constexpr int S = decltype(stage)::value;
    asm volatile("" ::: "memory");
    wait_loads(2 * kLoads * min(j1 - 1 - j, kStages - 2));
    lds_sync();
    fill(last, j + kStages - 1);
    compute(lds.k[S], lds.v[S], j, gr[S]);
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, (kStages > 2 ? 2 : 0)>;
  using S3 = std::integral_constant<int, (kStages > 2 ? 3 : 0)>;
  fill(S0{}, j0);
  if constexpr (kStages > 2) {
    fill(S1{}, j0 + 1);
    fill(S2{}, j0 + 2);
  }
  for (int j = j0; j < j1; j += kStages) {
    if constexpr (kStages == 2) {
      step(S0{}, S1{}, j);
      if (j + 1 < j1) step(S1{}, S0{}, j + 1);
    } else {
      step(S0{}, S3{}, j);
      if (j + 1 < j1) step(S1{}, S0{}, j + 1);
      if (j + 2 < j1) step(S2{}, S1{}, j + 2);
      if (j + 3 < j1) step(S3{}, S2{}, j + 3);
    }
  }

  l += lane_xor32(l);
  if (wrow + jq >= rows) return;
  // Without a maximum and a sum the row sees none of the range's keys, or scores that are all -inf: then there is
  // a page among those that it sees.
  bool seen = m > -INFINITY || l != 0.f;
  if (!seen) {
    const int none = min(j0, kb.na), some = min(j1, kb.na), from = max(j0 - kb.na, 0), to = max(j1 - kb.na, 0);
    const int part[2][2] = {{kTileKeys * (kb.a0 + none), kTileKeys * (kb.a0 + some)},
                            {kTileKeys * (kb.m0 + from), kTileKeys * (kb.m0 + to)}};
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {  // the first tokens and the rest, in either part of the list
      int key = max(max(k0, i & 2 ? lo : 0), i & 1 ? part[1][0] : part[0][0]);
      const int end = min(i & 2 ? hi : min(first, hi), i & 1 ? part[1][1] : part[0][1]);
#pragma unroll 1
      for (; key < end && !seen; key = (key / a.s.page_size + 1) * a.s.page_size)
        seen = (unsigned)table[key / a.s.page_size] < (unsigned)a.p.n_pages;
    }
  }
  if (direct) {
    const float inv = seen ? 1.f / l : 0.f;
    uint16_t* op = a.out + ((size_t)t * a.Hq + hq) * D + 4 * kh;
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<u32x2_t*>(op + 32 * d + 2 * r) =
            (u32x2_t){pack_bf16x2_rne(o[d][r] * inv, o[d][r + 1] * inv),
                      pack_bf16x2_rne(o[d][r + 2] * inv, o[d][r + 3] * inv)};
  } else {
    const size_t pr = (kShared ? (size_t)split * a.s.T + t : (size_t)(slot + (long long)split * sp.nn + tok)) * a.Hq + hq;
    float* op = (kShared ? a.shpart : a.opart) + pr * D + 4 * kh;
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4_t*>(op + 32 * d + 2 * r) =
            f32x4_t{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    if (kh == 0)
      *reinterpret_cast<float2*>((kShared ? a.shml : a.ml) + 2 * pr) = make_float2(seen_max(m * c, seen), l);
  }
  // (also where the result is final, so that the merge does not read an older launch's entry)
  if (!kShared && a.rows && split == 0 && hq == 0 && kh == 0)
    a.rows[t] = make_int4((int)(slot + tok), sp.nn, splits, 0);
}

// The launch: workgroups of the shared keys first (kWithShared), then those of the sequences' own keys. Both in
// one launch, since either alone leaves CUs idle.
template <int D, bool kOne, bool kWithShared>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PagedArgs a) {
  constexpr int kArr = kTileKeys * D, kFour = ring_stages<D>() > 2 ? kArr : 8;
  __shared__ __align__(16) uint16_t k0[kArr], v0[kArr], k1[kArr], v1[kArr], k2[kFour], v2[kFour], k3[kFour], v3[kFour];
  __shared__ float red[2][kOneWaves][16];
  __shared__ SharedRows sh;
  const Ring lds{{k0, k1, k2, k3}, {v0, v1, v2, v3}};
  int id = blockIdx.x;
  if constexpr (kWithShared) {
    if (id < a.sh_grid) {
      tile_body<D, true>(a, id / a.Hk, id % a.Hk, lds, sh);
      return;
    }
    id -= a.sh_grid;
  }
  if constexpr (kOne)
    one_body<D>(a, id / a.Hk, id % a.Hk, lds, red);
  else
    tile_body<D, false>(a, id / a.Hk, id % a.Hk, lds, sh);
}

// ------------------------------------------------------------------ merge of the partials
// kWavesPer waves per (token, head), or one wave per `per` heads of a token; lane = D / 64 dimensions. A partial
// without keys has maximum -inf. Bound by latency: 3.3 to 4.8 us for 12 to 1500 workgroups.
template <int D, int kWavesPer>
__global__ void __launch_bounds__(kWavesPer > 1 ? 64 * kWavesPer : 256) paged_merge_kernel(PagedArgs a, int per) {
  constexpr int V = D / 64, kBatch = 8, kRowsPer = kWavesPer > 1 ? 1 : 4;
  __shared__ float red_m[kWavesPer], red_l[kWavesPer], red_o[kWavesPer][D];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = a.Hq / per;
  const long long id = (long long)blockIdx.x * kRowsPer + wv / kWavesPer;
  const int t = __builtin_amdgcn_readfirstlane((int)(id / groups));
  const int h0 = __builtin_amdgcn_readfirstlane((int)(id % groups)) * per;
  const int w = wv % kWavesPer;
  bool live = t < a.s.T && (!a.s.q_start || (t >= a.s.q_start[0] && t < a.s.q_start[a.s.B]));
  int4 info = make_int4(0, 0, 0, 0);
  if (live) info = a.rows[t];
  // (a q_start that is not ascending can leave a row without this launch's entry: nothing out of range)
  live = live && info.x >= 0 && info.y > 0 && info.z > 0 &&
         info.x + (long long)info.y * (info.z - 1) < a.cap && (info.z > 1 || a.sh_splits > 0);
  const int parts = live ? a.sh_splits + info.z : 0;
  if (kWavesPer == 1 && !live) return;
  for (int h = h0; h < h0 + per; ++h) {
  float m = -INFINITY, l = 0.f, acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int p0 = w; p0 < parts; p0 += kWavesPer * kBatch) {
    float mv[kBatch], lv[kBatch], ov[kBatch][V];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int p = min(p0 + kWavesPer * u, parts - 1);
      const bool sh = p < a.sh_splits;
      const size_t row =
          (sh ? (size_t)p * a.s.T + t : (size_t)info.x + (size_t)info.y * (p - a.sh_splits)) * a.Hq + h;
      const float2 ml = *reinterpret_cast<const float2*>((sh ? a.shml : a.ml) + 2 * row);
      const float* op = (sh ? a.shpart : a.opart) + row * D + V * lane;
      mv[u] = p0 + kWavesPer * u < parts ? ml.x : -INFINITY;
      lv[u] = ml.y;
#pragma unroll
      for (int e = 0; e < V; ++e) ov[u][e] = op[e];
    }
    float mb = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, mv[u]);
    const float mz = mb == -INFINITY ? 0.f : mb;
    const float f0 = exp2f(m - mz);
    l *= f0;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= f0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = exp2f(mv[u] - mz);
      if (mv[u] > -INFINITY) {  // (a partial that counts nothing may repeat another's values)
        l = fmaf(f, lv[u], l);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(f, ov[u][e], acc[e]);
      }
    }
    m = mb;
  }
  if constexpr (kWavesPer > 1) {
    if (lane == 0) {
      red_m[wv] = m;
      red_l[wv] = l;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red_o[wv][V * lane + e] = acc[e];
    lds_sync();
    if (w != 0) return;
    float mt = red_m[0];
#pragma unroll
    for (int k = 1; k < kWavesPer; ++k) mt = fmaxf(mt, red_m[k]);
    const float mz = mt == -INFINITY ? 0.f : mt;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kWavesPer; ++k) {
      const float f = exp2f(red_m[k] - mz);
      l = fmaf(f, red_l[k], l);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(f, red_o[k][V * lane + e], acc[e]);
    }
    m = mt;
  }
  if (!live) return;
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  uint16_t* op = a.out + ((size_t)t * a.Hq + h) * D + V * lane;
  if constexpr (V == 2)
    *reinterpret_cast<uint32_t*>(op) = pack_bf16x2_rne(acc[0] * inv, acc[1] * inv);
  else
    *op = static_cast<uint16_t>(f32_to_bf16_rne(acc[0] * inv));
  }
}

// ------------------------------------------------------------------ launch plan
struct Plan {
  bool one;           // the one-token kernel
  int unit, target;   // least blocks per workgroup, workgroups aimed at
  long long items;    // workgroups per kv head of the own-keys launch
  long long ranges;   // of one sequence at most
  long long cap;      // token slots of the partials
  int sh_splits;
  long long sh_items;
  size_t bytes;       // workspace
};

bool sizes_ok(int T, int B, int Hq, int Hk, int D, int max_len, int shared) {
  return T > 0 && B > 0 && Hq > 0 && Hk > 0 && Hq % Hk == 0 && (D == 64 || D == 128) && max_len > 0 &&
         max_len < (1 << 30) && shared >= 0 && (long long)T * Hq < (1ll << 30) && B < (1 << 24);
}

Plan make_plan(int T, int B, int Hq, int Hk, int D, int max_len, bool ragged, int shared) {
  int cus = 256;  // (a failed query leaves MI355X's count; the launch reports the error)
  if (cached_cu_count(&cus) != hipSuccess || cus <= 0) cus = 256;
  Plan p{};
  const int R = Hq / Hk;
  shared = std::min(shared, max_len);
  // Token counts are device values, so with q_start single tokens go in tiles too. us without and with it (28 / 4
  // heads of 128; 14 / 2 of 64): one of 700 10.1, 15.1; 9.0, 13.3. 64 of 1000 to 8000 113, 146; 34, 60. 64 such
  // beside a prompt of 512 at 4000 184 in one call, 108 + 80 in two.
  p.one = !ragged && R <= 16;
  // Least range 64 keys (a block per wave) and 256. us with half, this and twice it: one token at 4000 13.2, 11.8,
  // 11.4; at 700 9.4, 9.5, 9.9; 20 tokens after 4000 19.4, 19.8, 23.8.
  p.unit = 4;
  // As many workgroups as run at once; tiles: one and a half per CU, since a range of few blocks costs a partial of
  // 128 rows (us with one, one and a half, two: 1000 tokens 42.3, 42.9, 49.5; 512 after 3000 68.1, 67.1, 59.8).
  p.target = p.one ? 2 * cus : 3 * cus / 2;
  if (shared > 0) {
    const long long st = ((long long)T * R + kTileRows - 1) / kTileRows;
    const int blocks = (shared + kTileKeys - 1) / kTileKeys;
    // One workgroup per CU, which leaves the other half of its LDS to the sequences' own keys. us for one, one and
    // a half, two and three, back to back: 96 sequences (194 tokens) behind 16384 99.6, 108.8, 116.5, 126.8.
    const long long want = cus / (st * Hk);
    // at least four blocks each, two where that leaves fewer than eight splits (8 sequences behind 1024: 14.4 ->
    // 11.8 us; always two: 32 behind 4096 23.3 -> 26.5)
    const int most = std::max(blocks / 4, std::min(blocks / 2, 8));
    p.sh_splits = (int)std::max(1ll, std::min<long long>(want, most));
    p.sh_items = st * p.sh_splits;
  }
  if (p.one && p.sh_items > 0)  // the rest of one round of workgroups
    p.target = (int)std::max<long long>(cus, 2ll * cus - p.sh_items * Hk);
  const int blk = p.one ? kOneRows : kTileKeys;
  const long long most = p.ranges = ((max_len + blk - 1) / blk + p.unit - 1) / p.unit;
  const long long tiles = p.one ? B : std::min<long long>((long long)T * R / kTileRows + B, (long long)T * R);
  const long long per_head = p.target / Hk + 2;
  p.items = std::min(tiles * most, per_head + tiles);
  p.cap = std::min((long long)T * most, T + (p.one ? 1 : kTileRows / R + 1) * per_head);
  if (p.cap > T || p.sh_splits > 0) {
    const size_t parts = ((size_t)p.cap + (size_t)p.sh_splits * T) * Hq;
    p.bytes = (size_t)T * sizeof(int4) + parts * (D + 2) * sizeof(float);
  }
  return p;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int D, bool kOne>
void launch_paged(const PagedArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.items * a.Hk + a.sh_grid));
  if (a.sh_grid > 0)
    hipLaunchKernelGGL((paged_attn_kernel<D, kOne, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_kernel<D, kOne, false>), grid, dim3(256), 0, st, a);
  if (p.bytes == 0) return;
  // Few rows with many partials (about that many, if the batch's sequences are alike) take a workgroup each: of
  // four waves, or of eight (us of the whole call with 1, 4, 8 and 16 waves: one sequence of 700, 11 partials,
  // 10.1, 9.4, 9.9, 10.5; 32 behind 4096 shared positions, 21 partials, 25.2, 22.8, 25.2, 30.5; one of 32000,
  // 129 partials, -, 23.3, 21.7, 21.7). Many rows, which seldom have more than one partial, take a wave per token.
  const long long rows = (long long)a.s.T * a.Hq;
  const long long most = p.sh_splits + std::min<long long>(p.target / ((long long)a.Hk * a.s.B) + 1, p.ranges);
  if (most > 64 && rows <= 8192) {
    hipLaunchKernelGGL((paged_merge_kernel<D, 8>), dim3((unsigned)rows), dim3(512), 0, st, a, 1);
  } else if (most > 8 && rows <= 8192) {
    hipLaunchKernelGGL((paged_merge_kernel<D, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, 1);
  } else {
    const int per = rows > 32768 ? a.Hq : 1;
    hipLaunchKernelGGL((paged_merge_kernel<D, 1>), dim3((unsigned)((rows / per + 3) / 4)), dim3(256), 0, st, a, per);
  }
}

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_paged_attention_workspace(int T, int B, int Hq, int Hk, int D, int max_len, int ragged,
                                    int shared) {
  if (!ns::sizes_ok(T, B, Hq, Hk, D, max_len, shared)) return 0;
  return ns::make_plan(T, B, Hq, Hk, D, max_len, ragged != 0, shared).bytes;
}

int ns_paged_attention(const void* q, long long q_stride, const void* k_pool, const void* v_pool,
                       long long page_stride, long long head_stride, int n_pages, int page_size,
                       const int* table, long long table_stride, int width, const int* lens,
                       const int* q_start, void* out, void* work, size_t work_bytes, int T, int B,
                       int Hq, int Hk, int D, int shared, int window, int sinks, float scale,
                       void* stream) {
  ns::PagedArgs a{};
  a.s = ns::Batch{q_start, lens, table, table_stride, T, B, width, page_size};
  a.p = ns::Pools{static_cast<uint16_t*>(const_cast<void*>(k_pool)),
                  static_cast<uint16_t*>(const_cast<void*>(v_pool)), page_stride, head_stride, n_pages};
  if (Hq <= 0 || Hk <= 0 || !ns::batch_ok(a.s, a.p, Hk, D)) return -2;
  const int max_len = width * page_size;
  if (!ns::sizes_ok(T, B, Hq, Hk, D, max_len, shared)) return -2;
  if (window < 0 || sinks < 0 || !(scale > 0.f) || !(scale < INFINITY)) return -2;
  if (!q || !out || !ns::aligned(q, 16) || !ns::aligned(out, 16)) return -2;
  if (q_stride % 8 || q_stride < (long long)Hq * D) return -2;
  const ns::Plan p = ns::make_plan(T, B, Hq, Hk, D, max_len, q_start != nullptr, shared);
  if ((p.items + p.sh_items) * Hk >= (1ll << 31) || p.cap >= (1ll << 31)) return -2;
  if (p.bytes > 0) {
    if (!work || !ns::aligned(work, 16) || work_bytes < p.bytes) return -2;
    a.rows = static_cast<int4*>(work);
    a.opart = reinterpret_cast<float*>(a.rows + T);
    a.shpart = a.opart + (size_t)p.cap * Hq * D;
    a.ml = a.shpart + (size_t)p.sh_splits * T * Hq * D;
    a.shml = a.ml + (size_t)p.cap * Hq * 2;
  }
  const ns::Bytes y = ns::bytes_of(out, 2 * (size_t)T * Hq * D), w = ns::bytes_of(p.bytes ? work : nullptr, p.bytes);
  for (const ns::Bytes r : {y, w}) {
    if (!ns::apart(r, ns::rows_of(q, T, q_stride, (long long)Hq * D, 2)) || !ns::metadata_apart(a.s, r)) return -2;
    for (const uint16_t* pool : {a.p.k, a.p.v})
      if (!ns::pool_apart(pool, a.p, Hk, (long long)page_size * D, r)) return -2;
  }
  if (!ns::apart(y, w)) return -2;
  a.cap = p.cap;
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<uint16_t*>(out);
  a.Hq = Hq;
  a.Hk = Hk;
  a.R = Hq / Hk;
  a.shared = std::min(shared, max_len);
  a.window = window;
  a.sinks = sinks;
  a.sh_splits = p.sh_splits;
  a.sh_grid = (int)(p.sh_items * Hk);
  a.unit = p.unit;
  a.per_target = (float)Hk / (float)p.target;
  a.c = scale * 1.4426950408889634f;
  const auto st = static_cast<hipStream_t>(stream);
  if (D == 64)
    p.one ? ns::launch_paged<64, true>(a, p, st) : ns::launch_paged<64, false>(a, p, st);
  else
    p.one ? ns::launch_paged<128, true>(a, p, st) : ns::launch_paged<128, false>(a, p, st);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
