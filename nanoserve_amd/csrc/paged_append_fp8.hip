// Bias, position rotation and append of a batch's new tokens to a paged KV cache held in 8 bits (contract in
// batch_ops.h): one launch for prompts and single tokens. No counterpart in the reference, whose cache is bf16.
//
// A block of 16 positions shares one power of two per kv head, so its new rows are taken together by one wave: rotated
// values in registers, the largest magnitude over the wave, then the codes. Where a block already holds rows and its
// exponent rises, the wave rewrites their codes too: a power of two moves e4m3's exponent alone, so that only values
// that leave the normal range are rounded again.
//  * With q_start: a wave per block, kv head and one of K and V; the query heads' workgroups behind them in the same launch, as
//    the blocks take longest. Bound by HBM: 4660 tokens (81 MB) 20.0 us, 4.06 TB/s of mixed reads and writes. K and V in one wave
//    23.7 us (151 registers), with the query heads first 28.4.
//  * One token per sequence: a thread group per head, whose loads do not wait for the length and the page. Bound by the chain
//    length -> page -> scale -> store: 16 tokens 4.1 us, the bf16 cache's append 3.9; with a wave per block 12.1.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "batch_ops.h"
#include "paged_common.h"

namespace ns {
namespace {

constexpr int kTile = 16;  // token rows whose blocks a workgroup finds together

struct Append8Args {
  const uint16_t *qkv, *bias;
  const float* inv_freq;
  uint16_t* q_out;
  long long qkv_stride;
  Batch s;
  Pools p;
  Scales f;
  int Hq, Hk;
  int kv_grid, parts;  // workgroups of the key and value heads, and how many of them per 16 token rows
};

// cos and sin of position * frequency, reduced to a fraction of a turn in fp64.
__device__ __forceinline__ void turn(int pos, float frq, float& sn, float& cs) {
  const double turns = (double)pos * ((double)frq * 0.15915494309189535);
  sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
}

// Elements 8 c .. + 7 of head h in a token's row, and their partners D / 2 further on, bias added.
template <int D>
__device__ __forceinline__ void load_pair(const Append8Args& a, const uint16_t* row, int h, int c, float (&x)[8],
                                          float (&y)[8]) {
  const int off = h * D + 8 * c;
  unpack8(*reinterpret_cast<const u32x4_t*>(row + off), x);
  unpack8(*reinterpret_cast<const u32x4_t*>(row + off + D / 2), y);
  if (a.bias) {
    float u[8], w[8];
    unpack8(*reinterpret_cast<const u32x4_t*>(a.bias + off), u);
    unpack8(*reinterpret_cast<const u32x4_t*>(a.bias + off + D / 2), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] += u[e];
      y[e] += w[e];
    }
  }
}

// Eight values / 2^e as codes; NaN and infinities as NaN.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float z[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float v = x[4 * i + k];
      z[k] = fabsf(v) <= FLT_MAX ? held448(v * inv) : __uint_as_float(0x7fc00000u);
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], c, true);
  }
  return make_uint2(w[0], w[1]);
}

// Sixteen codes times a power of two, rounded again where they leave the normal range.
__device__ __forceinline__ u32x4_t rescaled(u32x4_t v, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[i], true);
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(held448(lo[0] * f), held448(lo[1] * f), 0, false);
    v[i] = __builtin_amdgcn_cvt_pk_fp8_f32(held448(hi[0] * f), held448(hi[1] * f), w, true);
  }
  return v;
}

// The largest of a group of N lanes (4 or 8, aligned; values not negative), in all of them: DPP within rows of 16.
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
  auto from = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                                 0xf, 0xf, false));
  };
  v = fmaxf(v, from(v, std::integral_constant<int, 0xb1>{}));   // lane ^ 1
  v = fmaxf(v, from(v, std::integral_constant<int, 0x4e>{}));   // lane ^ 2
  if constexpr (N == 8) v = fmaxf(v, from(v, std::integral_constant<int, 0x141>{}));  // mirrored within 8
  return v;
}

// The largest of the wave's values, none below 0.
__device__ __forceinline__ float wave_top(float v) {
  v = lanes_max<8>(v);
  v = fmaxf(v, lane_xor8(v));
  v = fmaxf(v, lane_xor16(v));
  return fmaxf(v, lane_xor32(v));
}

// The codes of one of K and V for `count` new rows of a block behind `held` older ones. x, y: of the rows
// kRows * p + lane / kLanes.
template <int D, int kPasses>
__device__ __forceinline__ void store_block(uint8_t* block, uint8_t* scale, int held, int count, const float (&x)[kPasses][8],
                                            const float (&y)[kPasses][8]) {
  constexpr int kLanes = D / 16, kRows = kWave / kLanes;
  const int lane = __lane_id(), c = lane % kLanes, r = lane / kLanes;
  const int old = held > 0 ? *scale : 0;
  float top = 0.f;
#pragma unroll
  for (int p = 0; p < kPasses; ++p)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = fabsf(x[p][e]), v = fabsf(y[p][e]);
      if (kRows * p + r < count) top = fmaxf(top, fmaxf(u <= FLT_MAX ? u : 0.f, v <= FLT_MAX ? v : 0.f));
    }
  int e = scale_exponent(wave_top(top));
  if (held > 0) e = max(e, min(max(old - 127, kLeastScale), kMostScale));
  e = __builtin_amdgcn_readfirstlane(e);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = kRows * p + r;
    if (row < count) {
      uint8_t* dst = block + (held + row) * D + 8 * c;
      *reinterpret_cast<uint2*>(dst) = codes8(x[p], inv);
      *reinterpret_cast<uint2*>(dst + D / 2) = codes8(y[p], inv);
    }
  }
  if (lane == 0) *scale = (uint8_t)(e + 127);
  if (held == 0 || e + 127 == old) return;
  // the rows from before, in units of the new scale
  const float f = ldexpf(1.f, old - 127 - e);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = kRows * p + r;
    if (row < held) {
      u32x4_t* at = reinterpret_cast<u32x4_t*>(block + row * D + 16 * c);
      *at = rescaled(*at, f);
    }
  }
}

template <int D, int kHeads>
__global__ void __launch_bounds__(256) paged_append_fp8_kernel(Append8Args a) {
  constexpr int kLanes = D / 16, kRows = kWave / kLanes, kPasses = kTile / kRows;
  const int H = a.Hq;
  if ((int)blockIdx.x >= a.kv_grid) {
    // a thread: elements 8 c .. with their partners in up to kHeads query heads of a token
    const int nblk = (H + kHeads - 1) / kHeads;
    const long long id = (long long)(blockIdx.x - a.kv_grid) * 256 + threadIdx.x, tb = id / kLanes;
    if (tb / nblk >= a.s.T) return;
    const int c = (int)(id % kLanes), t = (int)(tb / nblk), h0 = (int)(tb % nblk) * kHeads;
    const int b = a.s.sequence(t);
    if (b < 0) return;
    int row0, nn;
    a.s.tokens(b, row0, nn);
    const int pos = a.s.positions(b) - nn + (t - row0);
    const uint16_t* row = a.qkv + (size_t)t * a.qkv_stride;
    float x[kHeads][8], y[kHeads][8], cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) load_pair<D>(a, row, min(h0 + i, H - 1), c, x[i], y[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) turn(pos, a.inv_freq[8 * c + e], sn[e], cs[e]);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (h0 + i >= H) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = x[i][e], q = y[i][e];
        x[i][e] = p * cs[e] - q * sn[e];
        y[i][e] = q * cs[e] + p * sn[e];
      }
      uint16_t* dst = a.q_out + ((size_t)t * H + h0 + i) * D + 8 * c;
      *reinterpret_cast<u32x4_t*>(dst) = pack8(x[i]);
      *reinterpret_cast<u32x4_t*>(dst + D / 2) = pack8(y[i]);
    }
    return;
  }
  // Blocks that begin among the workgroup's 16 token rows: those of a sequence's first new token or of a multiple of 16.
  // Every wave finds them all and takes its share of them times the kv heads.
  const int id = blockIdx.x, tile = id / a.parts;
  const int lane = __lane_id(), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = tile * kTile + (lane & 15);
  int page = -1, pos = -1, count = 0, at = 0;
  if (lane < kTile && t < a.s.T) {
    const int b = a.s.sequence(t);
    if (b >= 0) {
      int row0, nn;
      a.s.tokens(b, row0, nn);
      const int i = t - row0;
      pos = a.s.positions(b) - nn + i;
      if (pos >= 0 && (pos % kScaleRows == 0 || i == 0 || pos == 0)) {
        count = min(kScaleRows - pos % kScaleRows, nn - i);
        page = a.s.table[(size_t)b * a.s.table_stride + pos / a.s.page_size];
        at = pos % a.s.page_size;
      }
    }
  }
  unsigned long long todo = __ballot(count > 0 && (unsigned)page < (unsigned)a.p.n_pages);
  for (int n = 0; todo; todo &= todo - 1) {
    const int src = __builtin_ctzll(todo);
    for (int h = 0; h < 2 * a.Hk; ++h, ++n) {
      if (n % (4 * a.parts) != (id % a.parts) * 4 + wv) continue;
      const bool is_k = h < a.Hk;
      const int g = is_k ? h : h - a.Hk;
      const int rows = __builtin_amdgcn_readlane(count, src), p0 = __builtin_amdgcn_readlane(pos, src);
      const int in = __builtin_amdgcn_readlane(at, src), held = in % kScaleRows;
      const size_t pg = (size_t)__builtin_amdgcn_readlane(page, src);
      const size_t off = pg * a.p.page_stride + (size_t)g * a.p.head_stride + (size_t)(in - held) * D;
      const size_t soff = pg * a.f.page_stride + (size_t)g * a.f.head_stride + in / kScaleRows;
      const int c = lane % kLanes, r = lane / kLanes;
      float x[kPasses][8], y[kPasses][8];
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {  // (rows past the last repeat it, unstored)
        const uint16_t* row = a.qkv + (size_t)(tile * kTile + src + min(kRows * p + r, rows - 1)) * a.qkv_stride;
        load_pair<D>(a, row, a.Hq + h, c, x[p], y[p]);
      }
      if (is_k) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          if (kRows * p >= rows) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float sn, cs;
            turn(p0 + kRows * p + r, a.inv_freq[8 * c + e], sn, cs);
            const float k = x[p][e], v = y[p][e];
            x[p][e] = k * cs - v * sn;
            y[p][e] = v * cs + k * sn;
          }
        }
      }
      store_block<D, kPasses>(reinterpret_cast<uint8_t*>(is_k ? a.p.k : a.p.v) + off, (is_k ? a.f.k : a.f.v) + soff, held,
                              rows, x, y);
    }
  }
}

// One new token per sequence: a thread takes elements 8 c .. with their partners in one head of a token, D / 16 lanes a
// head, so the values' loads need not wait for the length and the page. Where a block's exponent rises, those lanes
// also rewrite its older rows.
template <int D>
__global__ void __launch_bounds__(256) paged_append_fp8_one_kernel(Append8Args a) {
  constexpr int kLanes = D / 16;
  const int H = a.Hq + 2 * a.Hk;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, th = id / kLanes;
  if (th / H >= a.s.T) return;  // (whole groups of kLanes lanes)
  const int c = (int)(id % kLanes), b = (int)(th / H), h = (int)(th % H);
  const int pos = a.s.positions(b) - 1;
  float x[8], y[8], frq[8];
  load_pair<D>(a, a.qkv + (size_t)b * a.qkv_stride, h, c, x, y);
#pragma unroll
  for (int e = 0; e < 8; ++e) frq[e] = a.inv_freq[8 * c + e];
  const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hk;
  const int g = h - a.Hq - (is_k ? 0 : a.Hk);
  int page = -1;
  if (!is_q && pos >= 0) page = a.s.table[(size_t)b * a.s.table_stride + pos / a.s.page_size];
  const bool stored = (unsigned)page < (unsigned)a.p.n_pages;
  const int at = max(pos, 0) % a.s.page_size, held = at % kScaleRows;
  uint8_t* scale = nullptr;
  int old = 0;
  if (stored) {
    scale = (is_k ? a.f.k : a.f.v) + (size_t)page * a.f.page_stride + (size_t)g * a.f.head_stride + at / kScaleRows;
    if (held > 0) old = *scale;
  }
  if (h < a.Hq + a.Hk) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float sn, cs;
      turn(pos, frq[e], sn, cs);
      const float p = x[e], q = y[e];
      x[e] = p * cs - q * sn;
      y[e] = q * cs + p * sn;
    }
  }
  if (is_q) {
    uint16_t* dst = a.q_out + ((size_t)b * a.Hq + h) * D + 8 * c;
    *reinterpret_cast<u32x4_t*>(dst) = pack8(x);
    *reinterpret_cast<u32x4_t*>(dst + D / 2) = pack8(y);
  }
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = fabsf(x[e]), v = fabsf(y[e]);
    top = fmaxf(top, fmaxf(u <= FLT_MAX ? u : 0.f, v <= FLT_MAX ? v : 0.f));
  }
  top = lanes_max<kLanes>(top);
  if (!stored) return;
  int e = scale_exponent(top);
  if (held > 0) e = max(e, min(max(old - 127, kLeastScale), kMostScale));
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  uint8_t* block = reinterpret_cast<uint8_t*>(is_k ? a.p.k : a.p.v) + (size_t)page * a.p.page_stride +
                   (size_t)g * a.p.head_stride + (size_t)(at - held) * D;
  uint8_t* dst = block + held * D + 8 * c;
  *reinterpret_cast<uint2*>(dst) = codes8(x, inv);
  *reinterpret_cast<uint2*>(dst + D / 2) = codes8(y, inv);
  if (c == 0) *scale = (uint8_t)(e + 127);
  if (held == 0 || e + 127 == old) return;
  const float f = ldexpf(1.f, old - 127 - e);
  u32x4_t v[kScaleRows - 1];
#pragma unroll
  for (int r = 0; r < kScaleRows - 1; ++r)
    if (r < held) v[r] = *reinterpret_cast<const u32x4_t*>(block + r * D + 16 * c);
#pragma unroll
  for (int r = 0; r < kScaleRows - 1; ++r)
    if (r < held) *reinterpret_cast<u32x4_t*>(block + r * D + 16 * c) = rescaled(v[r], f);
}

template <int D>
void launch_one(const Append8Args& a, hipStream_t st) {
  const long long threads = a.s.T * (a.Hq + 2ll * a.Hk) * (D / 16);
  hipLaunchKernelGGL(paged_append_fp8_one_kernel<D>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
}

template <int D, int kHeads>
void launch(Append8Args& a, hipStream_t st) {
  const long long nblk = (a.Hq + kHeads - 1) / kHeads, threads = a.s.T * nblk * (D / 16);
  const long long tiles = (a.s.T + kTile - 1) / kTile;
  // about one block and head to a wave: a tile of 16 rows begins one block or two, and one more for each sequence
  const long long blocks = std::min<long long>(kTile, 1 + (long long)kTile * a.s.B / a.s.T);
  a.parts = (int)((blocks * 2 * a.Hk + 3) / 4);
  a.kv_grid = (int)(tiles * a.parts);
  hipLaunchKernelGGL((paged_append_fp8_kernel<D, kHeads>), dim3((unsigned)(a.kv_grid + (threads + 255) / 256)), dim3(256), 0,
                     st, a);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Up to this many chunks of query heads a thread takes one head, so that a short batch spreads over the GPU.
constexpr long long kSmall = 65536;

}  // namespace
}  // namespace ns

extern "C" int ns_paged_append_fp8(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq,
                                   const int* q_start, const int* lens, const int* table, long long table_stride,
                                   int width, void* k_pool, void* v_pool, long long page_stride,
                                   long long head_stride, void* k_scales, void* v_scales,
                                   long long scale_page_stride, long long scale_head_stride, int n_pages,
                                   int page_size, void* q_out, int T, int B, int Hq, int Hk, int D, void* stream) {
  if (Hq <= 0 || Hk <= 0 || Hq > (1 << 16) || Hk > (1 << 16) || (D != 64 && D != 128)) return -2;
  ns::Append8Args a{};
  a.s = ns::Batch{q_start, lens, table, table_stride, T, B, width, page_size};
  a.p = ns::Pools{static_cast<uint16_t*>(k_pool), static_cast<uint16_t*>(v_pool), page_stride, head_stride, n_pages, 1};
  a.f = ns::Scales{static_cast<uint8_t*>(k_scales), static_cast<uint8_t*>(v_scales), scale_page_stride,
                   scale_head_stride};
  if (!ns::batch_ok(a.s, a.p, Hk, D) || !ns::scales_ok(a.f, a.p, Hk, page_size)) return -2;
  if (!qkv || !inv_freq || !q_out) return -2;
  if (!ns::aligned(qkv, 16) || !ns::aligned(bias, 16) || !ns::aligned(inv_freq, 4) || !ns::aligned(q_out, 16))
    return -2;
  if (qkv_stride % 8 || qkv_stride < (Hq + 2ll * Hk) * D) return -2;
  const long long head = (long long)page_size * D, marks = page_size / ns::kScaleRows;
  const ns::Pools f = ns::scale_pools(a.f, n_pages);
  const ns::Bytes x = ns::rows_of(qkv, T, qkv_stride, (Hq + 2ll * Hk) * D, 2),
                  y = ns::bytes_of(q_out, 2 * (size_t)T * Hq * D), w = ns::bytes_of(bias, 2 * (Hq + 2ull * Hk) * D),
                  z = ns::bytes_of(inv_freq, 2 * (size_t)D);
  for (const ns::Bytes r : {x, y, w, z, ns::lens_of(a.s), ns::starts_of(a.s), ns::table_of(a.s)})
    if (!ns::pool_apart(a.p.k, a.p, Hk, head, r) || !ns::pool_apart(a.p.v, a.p, Hk, head, r) ||
        !ns::pool_apart(f.k, f, Hk, marks, r) || !ns::pool_apart(f.v, f, Hk, marks, r))
      return -2;
  if (!ns::apart(y, x) || !ns::apart(y, w) || !ns::apart(y, z)) return -2;
  if (!ns::pools_apart(a.p, Hk, head) || !ns::pools_apart(f, Hk, marks) || !ns::metadata_apart(a.s, y)) return -2;
  for (const uint16_t* pool : {a.p.k, a.p.v})
    for (const uint16_t* scales : {f.k, f.v})
      if (!ns::sets_apart(pool, a.p, head, scales, f, marks, Hk)) return -2;
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.bias = static_cast<const uint16_t*>(bias);
  a.inv_freq = static_cast<const float*>(inv_freq);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.qkv_stride = qkv_stride;
  a.Hq = Hq;
  a.Hk = Hk;
  // (both parts of the grid within 2^30 workgroups)
  if ((long long)T * Hq * (D / 16) >= (1ll << 38) || (long long)T * Hk >= (1ll << 29)) return -2;
  const auto st = static_cast<hipStream_t>(stream);
  if (!q_start) {
    if ((long long)T * (Hq + 2ll * Hk) * (D / 16) >= (1ll << 38)) return -2;
    D == 64 ? ns::launch_one<64>(a, st) : ns::launch_one<128>(a, st);
    return static_cast<int>(hipGetLastError());
  }
  const bool small = (long long)T * Hq * (D / 16) <= ns::kSmall;
  if (D == 64)
    small ? ns::launch<64, 1>(a, st) : ns::launch<64, 4>(a, st);
  else
    small ? ns::launch<128, 1>(a, st) : ns::launch<128, 4>(a, st);
  return static_cast<int>(hipGetLastError());
}
