// Attention of a batch's new tokens over a paged KV cache (gfx950; contract in batch_ops.h): single
// tokens, prompts, a window with first tokens, and a prefix that all sequences share. The reference
// has PyTorch SDPA over one contiguous cache (python/nanoserve/qwen.py:124-133).
//
// Two launches at most: the keys of the shared prefix (tiles over all tokens' rows) together with each
// sequence's own keys (streamed for single tokens, else tiles), and a merge of the fp32 partials.
#include "paged_attn_common.h"

namespace ns {
namespace {

constexpr int kOneRows = 16;  // cache rows per block of the one-token kernel

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

  one_finish<D>(a, lds, red, o, m, l, b, g, split, slot, sp.splits, direct);
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

template <int D, bool kOne>
void launch_paged(const PagedArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.items * a.Hk + a.sh_grid));
  if (a.sh_grid > 0)
    hipLaunchKernelGGL((paged_attn_kernel<D, kOne, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_kernel<D, kOne, false>), grid, dim3(256), 0, st, a);
  launch_merge<D>(a, p, st);
}

}  // namespace
}  // namespace ns

extern "C" {

size_t ns_paged_attention_workspace(int T, int B, int Hq, int Hk, int D, int max_len, int ragged,
                                    int shared) {
  if (!ns::sizes_ok(T, B, Hq, Hk, D, max_len, shared)) return 0;
  return ns::make_plan(T, B, Hq, Hk, D, max_len, ragged != 0, shared, ns::kOneRows).bytes;
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
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<uint16_t*>(out);
  ns::Plan p;
  if (!ns::plan_call(a, p, work, work_bytes, Hq, Hk, D, shared, window, sinks, scale, ns::kOneRows)) return -2;
  const auto st = static_cast<hipStream_t>(stream);
  if (D == 64)
    p.one ? ns::launch_paged<64, true>(a, p, st) : ns::launch_paged<64, false>(a, p, st);
  else
    p.one ? ns::launch_paged<128, true>(a, p, st) : ns::launch_paged<128, false>(a, p, st);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
