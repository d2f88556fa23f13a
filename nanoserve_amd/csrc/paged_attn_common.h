// What the attention kernels over a paged cache share, whatever the cache holds (contract in batch_ops.h): how work
// is dealt out, the tiles of query rows, the merge of partials and the launch plan. paged_attn.hip: keys and values in
// bf16; paged_attn_fp8.hip: in e4m3 with a power of two per 16 positions and kv head.
//
// Work is dealt out on the device, because lengths are device values (a captured graph replays at any
// lengths): every workgroup adds up the key blocks of the whole batch, takes the share per workgroup
// that spreads them over `target` workgroups, and finds its own sequence, row tile and range of blocks
// by a wave-wide prefix sum over the sequences. One long and fifteen short sequences then end together.
#pragma once
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
constexpr int kOneWaves = 4;
// Where a row's largest logit (base 2) is larger, the maximum is taken off its scores before they are multiplied: s c - m c as
// one fma is off by m c's rounding, 2^-24 of it, by which all of the row's exponentials are moved together (2^-4 in the
// exponent up to here), and past 2^31 out of fp32.
constexpr float kFarLogit = 1048576.f;
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
  Scales f;          // of a cache in 8 bits
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

// Item `item` of the batch: its sequence, the number within it, and the sequence's first partial (a
// token slot). False past the last item. Uniform over the workgroup's waves. kSorted: up to 64 sequences go by falling
// length, so that what starts last is short.
template <int BLK, int ROWS, bool kSorted = false>
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
  // Tiles of a cache in 8 bits: half as many workgroups aimed at (one per CU) where the tiles times kv heads are nearly as
  // many as the two per CU, so that splitting them makes a second round, and from four fifths of one per CU on where the tiles'
  // lists are so short (in the mean) that a range costs more in partials than it gains. us with all and half of them, 28 / 4
  // heads of 128 on 256 CUs, by tiles times kv heads: 448 (8 x 200 to 300 tokens up to 1000 to 4000 positions) 209, 157; 392
  // (7 of the same, 39 blocks) 168, 136; 220 (1000 tokens, 16) 48.4, 44.4; 224 (4 x 250 tokens after 1000, 20) 60.8, 52.4; 256
  // (64 x 2 to 5 after 300 to 500, 6) 30.7, 28.0. Not halved: 256 (64 x 2 to 5 after 4000 to 8000, 94) 157, 237; 224 (4 x
  // 250 after 8000, 127) 207, 237; 220 (1000 after 30000, 477) 669, 826; 400 (100 x 2 to 5 after 4000 to 8000, 94) 269, 301.
  // Against the rule, by a few per cent: 256 (64 x 2 to 5 after 600 to 1000, 13) 39.6, 41.8; 224 (4 x 250 after 1500, 28)
  // 71.7, 66.0. Past 512 it makes little difference.
  float per_target = a.per_target;
  if constexpr (kSorted) {
    const float all = wave_sum(tiles), fill = all * per_target;
    if (fill > 0.8f || (fill > 0.4f && total <= (fill > 0.7f ? 60.f : 20.f) * all)) per_target *= 2.f;
  }
  const int share = __builtin_amdgcn_readfirstlane((int)ceilf(total * per_target));
  int per = max(a.unit, (share + a.unit - 1) / a.unit * a.unit);
  // Sequences end inside a share: where that makes more items than workgroups aimed at, the last ones would
  // start when the others end. Larger shares then, a few times at most, if the items can be that few at all
  // (us without and with: 64 sequences of 1000 to 8000 positions 118.7, 110.0; 20 of 1000 to 4000 with 8 kv
  // heads 41.9, 38.5; 200 of up to 1000, whose 800 items are more anyway, 51.6, 59.0).
  const bool fits = B <= 4 * kWave && wave_sum(tiles) * per_target < 0.9f;
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
    const float over = (float)__builtin_amdgcn_readlane(wave_scan(items), kWave - 1) * per_target;
    if (over <= 1.f) break;
    per = ((int)((float)per * fminf(over, 2.f)) / a.unit + 1) * a.unit;
  }

  int from = lane;  // the lane's sequence
  if (kSorted && B > 1 && B <= kWave) {
    int rank = 0;
    for (int i = 0; i < B; ++i) {
      const int other = __builtin_amdgcn_readlane(x.blocks, i);
      rank += (other > x.blocks) | ((other == x.blocks) & (i < lane));
    }
    // (lanes past the last sequence keep their place)
    from = __builtin_amdgcn_ds_permute(4 * (lane < B ? rank : lane), lane);
    x.n = __builtin_amdgcn_ds_bpermute(4 * from, x.n);
    x.row0 = __builtin_amdgcn_ds_bpermute(4 * from, x.row0);
    x.nn = __builtin_amdgcn_ds_bpermute(4 * from, x.nn);
    x.tiles = __builtin_amdgcn_ds_bpermute(4 * from, x.tiles);
    x.blocks = __builtin_amdgcn_ds_bpermute(4 * from, x.blocks);
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
      b = kSorted && B <= kWave ? __builtin_amdgcn_readlane(from, src) : base + src;
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

// The end of the one-token kernels: merge of the waves through their (then free) first stages, fp32, heads 0 .. 7
// in the K half and 8 .. 15 in the V half. o: heads 4 grp + r at dim 16 d + r16 of a wave; m, l: of head r16.
template <int D>
__device__ __forceinline__ void one_finish(const PagedArgs& a, const Ring& lds, float (&red)[2][kOneWaves][16],
                                           const f32x4_t (&o)[D / 16], float m, float l, int b, int g, int split,
                                           long long slot, int splits, bool direct) {
  constexpr int kBlk = 16 * D;  // a wave's part of a stage, in units of 2 bytes
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, grp = lane >> 4, R = a.R;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  if (a.rows && split == 0 && g == 0 && tid == 0) a.rows[b] = make_int4((int)slot, 1, splits, 0);
}

// ------------------------------------------------------------------ caches in 8 bits
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ i32x8_t join(const u32x4_t& a, const u32x4_t& b) {
  return (i32x8_t){(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// The scales of the 16 rows of a page and head that hold position `key`, K's in bits 0 .. 7 and V's in 8 .. 15; one for
// what is no page. 255, no power of two and never written by an append, counts as the one below it: rows that
// nobody sees are zeros times their scale. `landed` waits for the value: without it the compiler would wait at every
// use, behind the ring's loads.
constexpr int kNoScales = 127 | 127 << 8;
__device__ __forceinline__ void landed(int& s) { asm volatile("" : "+v"(s)); }
__device__ __forceinline__ int group_scales(const PagedArgs& a, int id, int g, int key) {
  int s = kNoScales;
  if ((unsigned)id < (unsigned)a.p.n_pages) {
    const size_t at = (size_t)id * a.f.page_stride + (size_t)g * a.f.head_stride + key % a.s.page_size / kScaleRows;
    s = min((int)a.f.k[at], 254) | min((int)a.f.v[at], 254) << 8;
  }
  return s;
}

// Eight codes as bf16, exact: the first four times one scale, the others times another (powers of two).
__device__ __forceinline__ bf16x8_t f8_values(u32x2_t x, float s0, float s1) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float s = i ? s1 : s0;
    v[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[i], s, false));
    v[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x[i], s, true));
  }
  return __builtin_bit_cast(bf16x8_t, v);
}

// ds_read_b64_tr_b8: the 16 lanes of a group read 8 rows of 16 bytes, lane l half l % 2 of row l / 2, and lane l
// receives byte l of each row, in order.
__device__ __forceinline__ u32x2_t lds_read_tr8(const uint16_t* p) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                         (__attribute__((address_space(3))) i32x2_t*)const_cast<uint16_t*>(p)));
}

// The bits of the four lanes of a quad together.
__device__ __forceinline__ int quad_or(int v) {
  v |= __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false);
  return v | __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false);
}

// s + A B for 32 keys and 32 queries over 64 dims of e4m3, with a power of two per row of either: bytes 2 `ka` of
// ks and `qa` of qs.
__device__ __forceinline__ f32x16_t scaled_product(const i32x8_t& k, const i32x8_t& q, const f32x16_t& s, int ka, int ks,
                                                   int qa, int qs) {
  if (ka == 0)
    return qa == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q, s, 0, 0, 0, ks, 0, qs)
                   : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q, s, 0, 0, 0, ks, 1, qs);
  return qa == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q, s, 0, 0, 2, ks, 0, qs)
                 : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, q, s, 0, 0, 2, ks, 1, qs);
}

// A query head's values as two e4m3 terms, x = 2^e (hi + lo / 16). bf16 has the 8 significant bits of two
// e4m3: lo, what hi's rounding left times 16, is at most 8 of its units, so the terms are exact for values down to 2^-14 of
// the head's largest, and within 2^-22 of that below. NaN and infinities become NaN.
// The head's exponent e; a lane holds N * 8 of the values (bf16), the lanes l ^ 32 (and l ^ 16, kOver16) the others.
template <int N, bool kOver16>
__device__ __forceinline__ int query_exponent(const u32x4_t (&q)[N]) {
  uint32_t top = 0;  // of the magnitudes, as bf16 bits << 16; infinities and NaN do not count
#pragma unroll
  for (int s = 0; s < N; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = (i & 1 ? q[s][i / 2] : q[s][i / 2] << 16) & 0x7fff0000u;
      top = max(top, m < 0x7f800000u ? m : 0u);
    }
  float t = __uint_as_float(top);
  t = fmaxf(t, lane_xor32(t));
  if constexpr (kOver16) t = fmaxf(t, lane_xor16(t));
  return scale_exponent(t);
}

// Eight of the values.
__device__ __forceinline__ void query_terms(const u32x4_t& q, int e, u32x2_t& hi, u32x2_t& lo) {
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  auto fit = [&](uint32_t bits) {
    return (bits & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : held448(__uint_as_float(bits) * inv);
  };
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t h = 0, l = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = fit(q[2 * w + i] << 16), y = fit(q[2 * w + i] & 0xffff0000u);
      const int b = __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false);
      const auto back = __builtin_amdgcn_cvt_pk_f32_fp8(b, false);
      const int r = __builtin_amdgcn_cvt_pk_fp8_f32((x - back[0]) * 16.f, (y - back[1]) * 16.f, 0, false);
      h |= (uint32_t)(b & 0xffff) << (16 * i);
      l |= (uint32_t)(r & 0xffff) << (16 * i);
    }
    hi[w] = h;
    lo[w] = l;
  }
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
// In 8 bits (kF8; paged_attn_fp8.hip): the scores on v_mfma_scale_f32_32x32x64_f8f6f4, codes as they lie in the cache with their
// scale bytes as operands, queries in two e4m3 terms; the values' codes by ds_read_b64_tr_b8, each wave turning what it
// reads into bf16 (64 instructions a block beside 40 products; a tile in bf16 that all waves share would save 48 of them for a
// barrier, LDS writes and twice the reads). A stage is half as large.
// Measured in bf16 (28 / 4 heads of 128): prompts of 5 sequences of 2000 to 8000 654 us, 677 TFLOP/s, with the second term
// 1015 (a large library product: 1265); matrix cores busy in half of the cycles and vector units in 58 %, at 1.8 GHz,
// so that products and softmax still take turns for much of the time. Issuing one half block's softmax between the
// products of its neighbours did not help (659 -> 681 to 730 us). 4095 tokens with a window of 1000 and 14 / 2 heads of
// 64 43 us. 96 drafts of 1 to 3 tokens behind 16384 shared positions 100 to 104 us back to back, 108 to 117 among
// other launches: 220 workgroups of the shared keys, one to a CU, with one wave per SIMD. In 8 bits: 604 us (732 TFLOP/s),
// 47.4 and 107, with one probability term 463, 41 and 94.
template <int D, bool kShared, bool kF8 = false>
__device__ __forceinline__ void tile_body(const PagedArgs& a, int item, int g, const Ring& lds, SharedRows& sh) {
  // (kRow: a row of the cache in units of 2 bytes)
  constexpr int kRow = kF8 ? D / 2 : D, kChunks = kRow / 8, kRowsPerLoad = 64 / kChunks, kLoads = 16 / kRowsPerLoad,
                kDT = D / 32, kStages = ring_stages<D>();
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
    if (!find_item<kTileKeys, kTileRows, kF8>(a, item, b, sp, within, slot)) return;
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

  // B operand of the scores: this lane's query at dims 16 s + 8 kh .. (8 bits: 64 s + 32 kh .., in two terms)
  u32x4_t qf[D / 16];
  int qe = 0;  // the exponents of the terms' scales, a byte each
  if constexpr (kF8) {
    const uint16_t* qp = a.q + (size_t)t * a.q_stride + (size_t)hq * D + 32 * kh;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(qp + 64 * (s / 4) + 8 * (s % 4));
    const int e = query_exponent<D / 16, false>(qf);
    qe = (e + 127) | (e - 4 + 127) << 8;
#pragma unroll
    for (int s = 0; s < D / 16; s += 4) {  // 32 values: two vectors of hi, two of lo
      u32x2_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) query_terms(qf[s + i], e, hi[i], lo[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qf[s + i] = (u32x4_t){hi[2 * i][0], hi[2 * i][1], hi[2 * i + 1][0], hi[2 * i + 1][1]};
        qf[s + 2 + i] = (u32x4_t){lo[2 * i][0], lo[2 * i][1], lo[2 * i + 1][0], lo[2 * i + 1][1]};
      }
    }
  } else {
    const uint16_t* qp = a.q + (size_t)t * a.q_stride + (size_t)hq * D + 8 * kh;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(qp + 16 * s);
  }

  // lane i: offset in the pools of 16-row group i % 4 of block j0 + 16 (.. / 16) + i / 4 of the list
  const int* table = a.s.table + (size_t)b * a.s.table_stride;
  uint64_t offs = 0, valid = 0;
  int k_scales = 0, v_scales = 0;  // of the four groups of the lane's block, a byte each
  auto refill = [&](int j) {
    const int v = j + (lane >> 2);
    int id = -1, key = 0;
    if (v < j1) {
      key = kTileKeys * kb.block(v) + 16 * (lane & 3);
      if (key < top) id = table[key / a.s.page_size];
      offs = (kF8 ? 1 : 2) * ((uint64_t)(uint32_t)id * a.p.page_stride + (uint64_t)g * a.p.head_stride +
                              (uint64_t)(key % a.s.page_size) * D);
    }
    valid = __ballot((unsigned)id < (unsigned)a.p.n_pages);
    if constexpr (kF8) {
      const int s = group_scales(a, id, g, key), at = 8 * (lane & 3);
      k_scales = quad_or((s & 0xff) << at);
      v_scales = quad_or((s >> 8) << at);
      landed(k_scales);
      landed(v_scales);
    }
  };
  // (16-byte chunks of a row lie in the order c ^ swz(row), so that the rows of one read hit distinct banks)
  auto k_swz = [](int r) { return kF8 ? (D == 128 ? (r >> 1) & 7 : (r >> 2) & 3) : D == 128 ? r & 15 : (r >> 1) & 7; };
  auto v_swz = [](int r) {
    return kF8 ? (D == 128 ? 2 * ((r >> 1 & 1) | (r >> 2 & 2)) : 2 * (r >> 3 & 1))
               : D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
  };
  uint32_t k_off[kLoads], v_off[kLoads];  // of this lane's 16 bytes in a group
  const int lr = lane / kChunks;
#pragma unroll
  for (int p = 0; p < kLoads; ++p) {
    const int r = kRowsPerLoad * p + lr;
    const uint32_t ch = lane % kChunks;
    k_off[p] = r * 2 * kRow + 16u * (ch ^ k_swz(16 * wv + r));
    v_off[p] = r * 2 * kRow + 16u * (ch ^ v_swz(r));
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
  auto issue = [&](uint16_t* ks, uint16_t* vs, int j, uint32_t& groups, int (&sc)[2]) {
    const int jj = j - j0;
    if ((jj & 15) == 0) refill(j);
    const int e = 4 * (jj & 15);
    groups = (uint32_t)(valid >> e) & 15u;
    if constexpr (kF8) {
      sc[0] = __builtin_amdgcn_readlane(k_scales, e);
      sc[1] = __builtin_amdgcn_readlane(v_scales, e);
    }
    const int key0 = kTileKeys * kb.block(j) + 16 * wv;
    uint32_t sees = 0xffffu;
    if constexpr (kShared)
      if (gaps) sees = seen16(key0);
    const bool ok = ((groups >> wv) & 1) != 0 && sees != 0;
    const uint64_t off = ok ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(offs >> 32), e + wv) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((uint32_t)offs, e + wv)
                            : 0;
    const auto kres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.k) + off, (short)0,
                                                        ok ? 32 * kRow : 0, 0x00020000);
    const auto vres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.v) + off, (short)0,
                                                        ok ? 32 * kRow : 0, 0x00020000);
#pragma unroll
    for (int p = 0; p < kLoads; ++p) attn_lds_load16(kres, &ks[16 * wv * kRow + 512 * p], k_off[p], 0);
    if (gaps ? sees == 0xffffu : key0 >= k0 && key0 >= low && key0 + 16 <= top) {
#pragma unroll
      for (int p = 0; p < kLoads; ++p) attn_lds_load16(vres, &vs[16 * wv * kRow + 512 * p], v_off[p], 0);
    } else {  // value rows that no row of the tile sees are zero, whatever the page holds
#pragma unroll
      for (int p = 0; p < kLoads; ++p) {
        const int key = key0 + kRowsPerLoad * p + lr;
        const bool see = gaps ? ((sees >> (key - key0)) & 1) != 0
                              : (key >= k0) & (key < top) & ((key >= low) | (key < first));
        attn_lds_load16(vres, &vs[16 * wv * kRow + 512 * p], see ? v_off[p] : kOut, 0);
      }
    }
  };

  f32x16_t o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, mc = 0.f, l = 0.f;
  bool far = false;  // some row's maximum is past kFarLogit
  const float c = a.c;

  // transpose-read offsets (in units of 2 bytes) of the 32-dim tiles at key row 4 kh + (lane % 16) / 4; 8 bits: at
  // the key rows of the probabilities' order, 4 kh .. + 3 and 8 + 4 kh .. + 3, two lanes to a row
  int vt[kDT];
  if constexpr (kF8) {
    const int i = lane & 15, rr = 4 * kh + ((i >> 1) & 3) + 8 * (i >> 3);
#pragma unroll
    for (int d = 0; d < kDT; ++d)
      vt[d] = rr * kRow + 8 * ((2 * d + ((lane >> 4) & 1)) ^ v_swz(rr)) + 4 * (lane & 1);
  } else {
    const int rr = 4 * kh + ((lane & 15) >> 2);
#pragma unroll
    for (int d = 0; d < kDT; ++d)
      vt[d] = rr * D + 8 * ((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swz(rr)) + 4 * (lane & 1);
  }

  auto compute = [&](const uint16_t* kt, const uint16_t* vb, int j, uint32_t groups, const int (&sc)[2]) {
    const int key0 = kTileKeys * kb.block(j);
    if (key0 >= hi_max || (key0 + kTileKeys <= lo_min && key0 >= first)) return;  // no row sees it
    f32x16_t s[2];
    // bytes 0 and 2: scales of this lane's key, of its group in the first 32 keys and in the second
    const int kscale = kF8 ? (int)((uint32_t)sc[0] >> (jq & 16 ? 8 : 0)) : 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
      if constexpr (kF8) {
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
          const int kr = 32 * u + jq;
          const u32x4_t k0 = *reinterpret_cast<const u32x4_t*>(&kt[kr * kRow + 8 * ((4 * d + 2 * kh) ^ k_swz(kr))]);
          const u32x4_t k1 = *reinterpret_cast<const u32x4_t*>(&kt[kr * kRow + 8 * ((4 * d + 2 * kh + 1) ^ k_swz(kr))]);
          const i32x8_t kf = join(k0, k1);
#pragma unroll
          for (int i = 0; i < 2; ++i)  // the query's terms
            s[u] = scaled_product(kf, join(qf[4 * d + 2 * i], qf[4 * d + 2 * i + 1]), s[u], u, kscale, i, qe);
        }
        continue;
      }
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
    if (far | __any(bm > m)) {
      const float mn = fmaxf(m, bm);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f((m - ms) * c);
      m = mn;
      mc = ms * c;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      far = __any(fabsf(mc) > kFarLogit);
      if (far) {
        mc = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] -= ms;
      }
    }
    u32x4_t pt[2][4];  // B operands of the four 16-key steps
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[u][r + 1], c, -mc));
        const uint32_t term = pack_bf16x2_rne(p0, p1);
        pt[0][2 * u + (r >> 3)][(r & 7) >> 1] = term;
        l += p0 + p1;
        pt[1][2 * u + (r >> 3)][(r & 7) >> 1] = pack_bf16x2_rne(p0 - __uint_as_float(term << 16),
                                                                p1 - __uint_as_float(term & 0xffff0000u));
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8_t vf[kDT];
      if constexpr (kF8) {
        const float scale = __uint_as_float(((uint32_t)sc[1] >> 8 * u & 0xffu) << 23);
#pragma unroll
        for (int d = 0; d < kDT; ++d) vf[d] = f8_values(lds_read_tr8(&vb[vt[d] + 16 * u * kRow]), scale, scale);
      }
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        if constexpr (kF8) break;
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
  int sg[kStages][2];
  auto fill = [&](auto stage, int j) {
    constexpr int S = decltype(stage)::value;
    if (j < j1) issue(lds.k[S], lds.v[S], j, gr[S], sg[S]);
  };
  auto step = [&](auto stage, auto last, int j) {
    constexpr int S = decltype(stage)::value;
    asm volatile("" ::: "memory");
    wait_loads(2 * kLoads * min(j1 - 1 - j, kStages - 2));
    lds_sync();
    fill(last, j + kStages - 1);
    compute(lds.k[S], lds.v[S], j, gr[S], sg[S]);
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

inline bool sizes_ok(int T, int B, int Hq, int Hk, int D, int max_len, int shared) {
  return T > 0 && B > 0 && Hq > 0 && Hk > 0 && Hq % Hk == 0 && (D == 64 || D == 128) && max_len > 0 &&
         max_len < (1 << 30) && shared >= 0 && (long long)T * Hq < (1ll << 30) && B < (1 << 24);
}

// one_rows: cache rows per block of the one-token kernel.
inline Plan make_plan(int T, int B, int Hq, int Hk, int D, int max_len, bool ragged, int shared, int one_rows,
                      bool fp8 = false) {
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
  p.target = p.one || fp8 ? 2 * cus : 3 * cus / 2;
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
  const int blk = p.one ? one_rows : kTileKeys;
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

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }


template <int D>
void launch_merge(const PagedArgs& a, const Plan& p, hipStream_t st) {
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

// A call's checks and plan, with a.s, a.p, a.q, a.q_stride and a.out filled in: the rest of a, or false.
inline bool plan_call(PagedArgs& a, Plan& p, void* work, size_t work_bytes, int Hq, int Hk, int D, int shared,
                      int window, int sinks, float scale, int one_rows) {
  if (Hq <= 0 || Hk <= 0 || !batch_ok(a.s, a.p, Hk, D)) return false;
  const int T = a.s.T, B = a.s.B, max_len = a.s.width * a.s.page_size;
  if (!sizes_ok(T, B, Hq, Hk, D, max_len, shared)) return false;
  if (window < 0 || sinks < 0 || !(scale > 0.f) || !(scale < INFINITY)) return false;
  if (!a.q || !a.out || !aligned(a.q, 16) || !aligned(a.out, 16)) return false;
  if (a.q_stride % 8 || a.q_stride < (long long)Hq * D) return false;
  p = make_plan(T, B, Hq, Hk, D, max_len, a.s.q_start != nullptr, shared, one_rows, a.p.size == 1);
  if ((p.items + p.sh_items) * Hk >= (1ll << 31) || p.cap >= (1ll << 31)) return false;
  if (p.bytes > 0) {
    if (!work || !aligned(work, 16) || work_bytes < p.bytes) return false;
    a.rows = static_cast<int4*>(work);
    a.opart = reinterpret_cast<float*>(a.rows + T);
    a.shpart = a.opart + (size_t)p.cap * Hq * D;
    a.ml = a.shpart + (size_t)p.sh_splits * T * Hq * D;
    a.shml = a.ml + (size_t)p.cap * Hq * 2;
  }
  const Bytes y = bytes_of(a.out, 2 * (size_t)T * Hq * D), w = bytes_of(p.bytes ? work : nullptr, p.bytes);
  for (const Bytes r : {y, w}) {
    if (!apart(r, rows_of(a.q, T, a.q_stride, (long long)Hq * D, 2)) || !metadata_apart(a.s, r)) return false;
    for (const uint16_t* pool : {a.p.k, a.p.v})
      if (!pool_apart(pool, a.p, Hk, (long long)a.s.page_size * D, r)) return false;
  }
  if (!apart(y, w)) return false;
  a.cap = p.cap;
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
  return true;
}

}  // namespace
}  // namespace ns
