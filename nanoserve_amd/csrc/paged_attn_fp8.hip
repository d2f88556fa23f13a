// Attention of a batch's new tokens over a paged KV cache held in 8 bits (gfx950; contract in batch_ops.h): e4m3
// codes with a power of two per 16 positions and kv head, K and V apart. The cases, the split of the work and the
// merge are those of the cache in bf16 (paged_attn_common.h).
//
//  * Scores: the query's 8 significant bits are exactly two e4m3 terms, so q . k runs on the 8-bit matrix
//    instructions with the codes as they lie in the cache, at the price of one product in bf16.
//  * Values: a code times its scale is a bf16 value without rounding (v_cvt_scalef32_pk_bf16_fp8, two per
//    instruction), and the second product is the bf16 cache's.
//  * Probabilities are two bf16 terms, as over the bf16 cache: a token has the same weights, to 16 bits, whether it comes alone
//    or in a tile. With one term in tiles prompts of 5 sequences of 2000 to 8000 take 467 us instead of 612; weights are then off
//    by 2^-9 each, which shows in full where values cancel, and the 2-norm error against 64 bits is 0.0019 instead of 0.0017.
#include "paged_attn_common.h"

namespace ns {
namespace {

constexpr int kOneRows = 32;  // cache rows per block of the one-token kernel: as many bytes as 16 in bf16

typedef long i64_t;

// ------------------------------------------------------------------ one token per sequence
// As the bf16 cache's kernel: up to 16 query heads per kv head, a workgroup per range of blocks of one sequence and kv
// head, every fourth block a wave's own, streamed through its ring of LDS stages. A block is two groups of 16 rows, each in
// one page with one scale.
//  * Scores: v_mfma_f32_16x16x32_fp8_fp8, K rows as the A operand, the heads' terms as columns; a lane then has four keys
//    of each group for one head. Dims go in the order in which 16-byte reads of a row deliver them.
//  * Values: v_mfma_f32_16x16x32_bf16 over the 32 keys in the order of the scores' registers; V by transposed
//    8-bit LDS reads.
//  * The first blocks' loads go out beside those of their scales, which depend on the page ids too (16 sequences 23.2 ->
//    22.9 us), and probabilities come from v_exp_f32 as it is (22.7 -> 22.1).
// Measured (28 / 4 heads of 128): 4 sequences of 98 000 72 us, 5.5 TB/s, the streaming launch 65.2 and 6.1; 16 of 33 to 8191
// 22.3 us, 18 before the merge; 32 with a window of 4096 32.7; 64 of 1000 to 8000 70 (4.3 TB/s: the longest range is a third
// above the mean one); one of 700 with 12 / 2 heads 11.0, the latency of length -> page -> scale and rows -> merge. Shares of
// equal size cut from all sequences end to end take 64 us there but 29 for 16 sequences and 23 for 64 of up to 100 (8.9), as a
// workgroup then starts on two sequences or more; three or four workgroups per CU aimed at 26.8 and 26.8 for the 16.
template <int D>
__device__ __forceinline__ void one8_body(const PagedArgs& a, int item, int g, const Ring& lds,
                                          float (&red)[2][kOneWaves][16]) {
  // (a row of the cache in units of 2 bytes)
  constexpr int kRow = D / 2, kBlk = kOneRows * kRow, kChunks = kRow / 8, kRowsPerLoad = 64 / kChunks,
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

  // lane i: offset in the pools, first position and scales of group i % 2 of the wave's block 32 (.. / 32) + i / 2;
  // no page: position -1
  const int* table = a.s.table + (size_t)b * a.s.table_stride;
  uint64_t offs = 0;
  int keys = -1, scales = kNoScales;
  auto refill = [&](int i) {
    const int v = i + (lane >> 1);
    int id = -1, key = 0;
    if (v < cnt) {
      key = kOneRows * kb.block(j0 + wv + kOneWaves * v) + 16 * (lane & 1);
      if (key < n) id = table[key / a.s.page_size];
      offs = (uint64_t)(uint32_t)id * a.p.page_stride + (uint64_t)g * a.p.head_stride +
             (uint64_t)(key % a.s.page_size) * D;
    }
    keys = (unsigned)id < (unsigned)a.p.n_pages ? key : -1;
    scales = group_scales(a, id, g, key);
  };

  // B operand of the scores: lane (head l % 16, grp = l / 16), dims 64 s + 16 grp ..; heads past R: 0
  const int r16 = lane & 15, grp = lane >> 4;
  u32x4_t qf[D / 32];
  {
    const uint16_t* qp = a.q + (size_t)b * a.q_stride + (size_t)(g * R + min(r16, R - 1)) * D + 16 * grp;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(qp + 64 * (s / 2) + 8 * (s % 2));
      qf[s] = r16 < R ? v : u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  if (cnt > 0) refill(0);  // (its loads beside the query's)
  i64_t qh[D / 32], ql[D / 32];
  const int qe = query_exponent<D / 32, true>(qf);
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    u32x2_t hi, low;
    query_terms(qf[s], qe, hi, low);
    qh[s] = __builtin_bit_cast(i64_t, hi);
    ql[s] = __builtin_bit_cast(i64_t, low);
  }

  auto k_swz = [](int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  auto v_swz = [](int row) {
    return D == 128 ? (row >> 1 & 3) | (row >> 4 & 1) << 2 : (row >> 2 & 1) | (row >> 4 & 1) << 1;
  };
  auto seen_key = [&](int key) { return (key < n) & (key >= k0) & ((key >= lo) | (key < first)); };
  uint32_t k_off[kLoads], v_off[kLoads];  // of this lane's 16 bytes in a group
  const int lr = lane / kChunks;
#pragma unroll
  for (int p = 0; p < kLoads; ++p) {
    const int row = kRowsPerLoad * p + lr;
    const uint32_t ch = lane % kChunks;
    k_off[p] = row % 16 * D + 16u * (ch ^ k_swz(row));
    v_off[p] = row % 16 * D + 16u * (ch ^ v_swz(row));
  }
  struct At {  // a block in flight: its first position, which groups have a page, their scales
    int key0, sc[2];
    bool has[2], whole;
  };
  auto issue = [&](uint16_t* ks, uint16_t* vs, int i, At& at) {
    if (i > 0 && (i & 31) == 0) {
      refill(i);
      landed(scales);
    }
    const int e = 2 * (i & 31);
    at.key0 = kOneRows * kb.block(j0 + wv + kOneWaves * i);
    at.whole = at.key0 >= k0 && at.key0 >= lo && at.key0 + kOneRows <= n;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (i >= kStages) at.sc[u] = __builtin_amdgcn_readlane(scales, e + u);
      at.has[u] = __builtin_amdgcn_readlane(keys, e + u) >= 0;
      at.whole &= at.has[u];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool ok = at.has[u];
      const uint64_t off = ok ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(offs >> 32), e + u) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((uint32_t)offs, e + u)
                              : 0;
      const auto kres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.k) + off, (short)0,
                                                          ok ? 16 * D : 0, 0x00020000);
      const auto vres = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>(a.p.v) + off, (short)0,
                                                          ok ? 16 * D : 0, 0x00020000);
#pragma unroll
      for (int p = u * kLoads / 2; p < (u + 1) * kLoads / 2; ++p) lds_stream16(kres, ks + 512 * p, k_off[p]);
      if (at.whole) {
#pragma unroll
        for (int p = u * kLoads / 2; p < (u + 1) * kLoads / 2; ++p) lds_stream16(vres, vs + 512 * p, v_off[p]);
      } else {
#pragma unroll
        for (int p = u * kLoads / 2; p < (u + 1) * kLoads / 2; ++p)
          lds_stream16(vres, vs + 512 * p, seen_key(at.key0 + kRowsPerLoad * p + lr) ? v_off[p] : kOut);
      }
    }
  };

  f32x4_t o[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // of head r16
  bool seen = false;             // a block of the wave had a page, and so a key that the token sees
  // row of a transposed read: the keys 4 grp .. + 3 of either group, two lanes to a row
  const int vrow = 4 * grp + ((r16 >> 1) & 3) + 16 * (r16 >> 3);
  auto compute = [&](const uint16_t* ks, const uint16_t* vs, const At& at) {
    float sr[2][4], bm = -INFINITY;  // head r16, keys 16 u + 4 grp + r (base-2 logits)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4_t hi = {0.f, 0.f, 0.f, 0.f}, low = {0.f, 0.f, 0.f, 0.f};
      const int row = 16 * u + r16;
#pragma unroll
      for (int s = 0; s < D / 64; ++s) {
        const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(ks + row * kRow + 8 * ((4 * s + grp) ^ k_swz(row)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const i64_t x = __builtin_bit_cast(i64_t, (u32x2_t){kf[2 * h], kf[2 * h + 1]});
          hi = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(x, qh[2 * s + h], hi, 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(x, ql[2 * s + h], low, 0, 0, 0);
        }
      }
      // (as an exponent: the powers of two of query and keys together may pass fp32 where the score is small or 0)
      const int e = qe + (at.sc[u] & 0xff) - 127;
#pragma unroll
      for (int r = 0; r < 4; ++r) sr[u][r] = __builtin_amdgcn_ldexpf(fmaf(low[r], 0.0625f, hi[r]), e) * a.c;
    }
    if (!at.whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sr[u][r] = at.has[u] & seen_key(at.key0 + 16 * u + 4 * grp + r) ? sr[u][r] : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) bm = fmaxf(bm, fmaxf(sr[0][r], sr[1][r]));
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
    u32x4_t ph, pl;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(sr[u][r] - mz), p1 = __builtin_amdgcn_exp2f(sr[u][r + 1] - mz);
        l += p0 + p1;  // this lane's keys; the lanes are added at the end
        const uint32_t term = pack_bf16x2_rne(p0, p1);
        ph[2 * u + r / 2] = term;
        pl[2 * u + r / 2] = pack_bf16x2_rne(p0 - __uint_as_float(term << 16), p1 - __uint_as_float(term & 0xffff0000u));
      }
    const float s0 = __uint_as_float((uint32_t)(at.sc[0] >> 8) << 23), s1 = __uint_as_float((uint32_t)(at.sc[1] >> 8) << 23);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const bf16x8_t vb = f8_values(lds_read_tr8(vs + vrow * kRow + 8 * (d ^ v_swz(vrow)) + 4 * (lane & 1)), s0, s1);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ph), vb, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pl), vb, o[d], 0, 0, 0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is read before it is loaded again
    asm volatile("" ::: "memory");
  };

  At at[kStages];  // the blocks in flight
  auto start = [&](auto stage, int i) {
    constexpr int S = decltype(stage)::value;
    issue(lds.k[S] + wv * kBlk, lds.v[S] + wv * kBlk, i, at[S]);
  };
  auto step = [&](auto stage, int i) {
    constexpr int S = decltype(stage)::value;
    wait_loads(2 * kLoads * min(cnt - 1 - i, kStages - 1));
    seen |= at[S].has[0] | at[S].has[1];
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
  landed(scales);  // (of the first refill: behind the first blocks' loads)
#pragma unroll
  for (int k = 0; k < kStages; ++k)
#pragma unroll
    for (int u = 0; u < 2; ++u) at[k].sc[u] = __builtin_amdgcn_readlane(scales, 2 * k + u);
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
  one_finish<D>(a, lds, red, o, m, l, b, g, split, slot, sp.splits, direct);
}

// The launch: workgroups of the shared keys first (kWithShared), then those of the sequences' own keys. Both in
// one launch, since either alone leaves CUs idle.
template <int D, bool kOne, bool kWithShared>
__global__ void __launch_bounds__(256, 2) paged_attn_fp8_kernel(PagedArgs a) {
  constexpr int kArr = kOne ? kTileKeys * D : kTileKeys * D / 2, kFour = ring_stages<D>() > 2 ? kArr : 8;
  __shared__ __align__(16) uint16_t k0[kArr], v0[kArr], k1[kArr], v1[kArr], k2[kFour], v2[kFour], k3[kFour], v3[kFour];
  __shared__ float red[2][kOneWaves][16];
  __shared__ SharedRows sh;
  const Ring lds{{k0, k1, k2, k3}, {v0, v1, v2, v3}};
  int id = blockIdx.x;
  if constexpr (kWithShared) {
    if (id < a.sh_grid) {
      tile_body<D, true, true>(a, id / a.Hk, id % a.Hk, lds, sh);
      return;
    }
    id -= a.sh_grid;
  }
  if constexpr (kOne)
    one8_body<D>(a, id / a.Hk, id % a.Hk, lds, red);
  else
    tile_body<D, false, true>(a, id / a.Hk, id % a.Hk, lds, sh);
}

template <int D, bool kOne>
void launch_paged(const PagedArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.items * a.Hk + a.sh_grid));
  if (a.sh_grid > 0)
    hipLaunchKernelGGL((paged_attn_fp8_kernel<D, kOne, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_fp8_kernel<D, kOne, false>), grid, dim3(256), 0, st, a);
  launch_merge<D>(a, p, st);
}

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_paged_attention_fp8_workspace(int T, int B, int Hq, int Hk, int D, int max_len, int ragged,
                                        int shared) {
  if (!ns::sizes_ok(T, B, Hq, Hk, D, max_len, shared)) return 0;
  return ns::make_plan(T, B, Hq, Hk, D, max_len, ragged != 0, shared, ns::kOneRows, true).bytes;
}

int ns_paged_attention_fp8(const void* q, long long q_stride, const void* k_pool, const void* v_pool,
                           long long page_stride, long long head_stride, const void* k_scales, const void* v_scales,
                           long long scale_page_stride, long long scale_head_stride, int n_pages, int page_size,
                           const int* table, long long table_stride, int width, const int* lens,
                           const int* q_start, void* out, void* work, size_t work_bytes, int T, int B,
                           int Hq, int Hk, int D, int shared, int window, int sinks, float scale,
                           void* stream) {
  ns::PagedArgs a{};
  a.s = ns::Batch{q_start, lens, table, table_stride, T, B, width, page_size};
  a.p = ns::Pools{static_cast<uint16_t*>(const_cast<void*>(k_pool)),
                  static_cast<uint16_t*>(const_cast<void*>(v_pool)), page_stride, head_stride, n_pages, 1};
  a.f = ns::Scales{static_cast<uint8_t*>(const_cast<void*>(k_scales)),
                   static_cast<uint8_t*>(const_cast<void*>(v_scales)), scale_page_stride, scale_head_stride};
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<uint16_t*>(out);
  ns::Plan p;
  if (!ns::plan_call(a, p, work, work_bytes, Hq, Hk, D, shared, window, sinks, scale, ns::kOneRows)) return -2;
  if (!ns::scales_ok(a.f, a.p, Hk, page_size)) return -2;
  const ns::Pools f = ns::scale_pools(a.f, n_pages);
  for (const ns::Bytes r : {ns::bytes_of(out, 2 * (size_t)T * Hq * D), ns::bytes_of(p.bytes ? work : nullptr, p.bytes)})
    for (const uint16_t* pool : {f.k, f.v})
      if (!ns::pool_apart(pool, f, Hk, page_size / ns::kScaleRows, r)) return -2;
  const auto st = static_cast<hipStream_t>(stream);
  if (D == 64)
    p.one ? ns::launch_paged<64, true>(a, p, st) : ns::launch_paged<64, false>(a, p, st);
  else
    p.one ? ns::launch_paged<128, true>(a, p, st) : ns::launch_paged<128, false>(a, p, st);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
