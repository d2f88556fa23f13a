// Bias, position rotation and append of a batch's new tokens to a paged KV cache (contract in
// batch_ops.h), one launch for prompts and single tokens alike. The reference does these for one
// sequence with PyTorch ops and its RoPE (python/nanoserve/qwen.py:119-122, 147-151).
//
// Bound by HBM for prompts (each value read once and written once) and by one chain of dependent loads
// for single tokens: length -> page -> store, with the loads of the values, the bias and the
// frequencies, and the angles' arithmetic, beside it. Thread (token, head block, chunk c) rotates elements 8c .. 8c + 7 with their partners D/2
// further on in up to kHeads heads, so the chunk's eight angles serve all of them.
//  * Angles: position * inv_freq in fp64, reduced to a fraction of a turn there, then sincospif in fp32
//    on [-1, 1]: at position 10^6 an fp32 product would be off by 0.03 radians.
#include <math.h>
#include <stdint.h>

#include "batch_ops.h"
#include "paged_common.h"

namespace ns {
namespace {


// Up to this many chunks a thread takes one head, so that a short batch spreads over the GPU; beyond it six heads
// share a thread's angles. us for one, two, three and six heads: 16 tokens of 36 heads 3.9, 4.4, 4.9, 6.5; 4660 tokens
// 25.8, 21.6, 20.9, 20.3 (of 86 MB, 4.2 TB/s).
constexpr long long kSmall = 65536;

struct AppendArgs {
  const uint16_t *qkv, *bias;
  const float* inv_freq;
  uint16_t* q_out;
  long long qkv_stride;
  Batch s;
  Pools p;
  int Hq, Hk, D;
};

template <int kHeads>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
  const int D = a.D, chunks = D >> 4, H = a.Hq + 2 * a.Hk, nblk = (H + kHeads - 1) / kHeads;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(id % chunks);
  const long long tb = id / chunks;
  if (tb / nblk >= a.s.T) return;
  const int t = (int)(tb / nblk), h0 = (int)(tb % nblk) * kHeads;
  // the metadata's loads go out first: the page's address waits for two of them in turn
  const int b = a.s.sequence(t);
  if (b < 0) return;
  int row0, nn;
  a.s.tokens(b, row0, nn);
  const int len = a.s.positions(b);
  const uint16_t* row = a.qkv + (size_t)t * a.qkv_stride;
  u32x4_t lo[kHeads], hi[kHeads], blo[kHeads], bhi[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int off = min(h0 + i, H - 1) * D + 8 * c;  // heads past H repeat the last, unstored
    lo[i] = *reinterpret_cast<const u32x4_t*>(row + off);
    hi[i] = *reinterpret_cast<const u32x4_t*>(row + off + D / 2);
    if (a.bias) {
      blo[i] = *reinterpret_cast<const u32x4_t*>(a.bias + off);
      bhi[i] = *reinterpret_cast<const u32x4_t*>(a.bias + off + D / 2);
    }
  }
  float frq[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) frq[e] = a.inv_freq[8 * c + e];

  const int pos = len - nn + (t - row0);
  const bool stored = pos >= 0 && h0 + kHeads > a.Hq;
  const int page = stored ? a.s.table[(size_t)b * a.s.table_stride + pos / a.s.page_size] : -1;

  float cs[8], sn[8];
  if (h0 < a.Hq + a.Hk) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double turns = (double)pos * ((double)frq[e] * 0.15915494309189535);
      sincospif((float)(2.0 * (turns - rint(turns))), &sn[e], &cs[e]);
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    if (h >= H) break;
    float x[8], y[8];
    unpack8(lo[i], x);
    unpack8(hi[i], y);
    if (a.bias) {
      float u[8], w[8];
      unpack8(blo[i], u);
      unpack8(bhi[i], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] += u[e];
        y[e] += w[e];
      }
    }
    if (h < a.Hq + a.Hk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = x[e], q = y[e];
        x[e] = p * cs[e] - q * sn[e];
        y[e] = q * cs[e] + p * sn[e];
      }
    }
    uint16_t* dst;
    if (h < a.Hq) {
      dst = a.q_out + ((size_t)t * a.Hq + h) * D;
    } else {
      if ((unsigned)page >= (unsigned)a.p.n_pages) continue;
      const bool is_k = h < a.Hq + a.Hk;
      dst = (is_k ? a.p.k : a.p.v) + (size_t)page * a.p.page_stride +
            (size_t)(h - a.Hq - (is_k ? 0 : a.Hk)) * a.p.head_stride + (size_t)(pos % a.s.page_size) * D;
    }
    *reinterpret_cast<u32x4_t*>(dst + 8 * c) = pack8(x);
    *reinterpret_cast<u32x4_t*>(dst + D / 2 + 8 * c) = pack8(y);
  }
}

template <int kHeads>
void launch_append(const AppendArgs& a, hipStream_t st) {
  const long long nblk = (a.Hq + 2ll * a.Hk + kHeads - 1) / kHeads, threads = a.s.T * nblk * (a.D / 16);
  hipLaunchKernelGGL(paged_append_kernel<kHeads>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace ns

extern "C" int ns_paged_append(const void* qkv, long long qkv_stride, const void* bias,
                               const void* inv_freq, const int* q_start, const int* lens,
                               const int* table, long long table_stride, int width, void* k_pool,
                               void* v_pool, long long page_stride, long long head_stride, int n_pages,
                               int page_size, void* q_out, int T, int B, int Hq, int Hk, int D,
                               void* stream) {
  if (Hq <= 0 || Hk <= 0 || Hq > (1 << 16) || Hk > (1 << 16) || D <= 0 || D % 16 || D > 512) return -2;
  ns::AppendArgs a{};
  a.s = ns::Batch{q_start, lens, table, table_stride, T, B, width, page_size};
  a.p = ns::Pools{static_cast<uint16_t*>(k_pool), static_cast<uint16_t*>(v_pool), page_stride,
                  head_stride, n_pages};
  if (!ns::batch_ok(a.s, a.p, Hk, D)) return -2;
  if (!qkv || !inv_freq || !q_out) return -2;
  if (!ns::aligned(qkv, 16) || !ns::aligned(bias, 16) || !ns::aligned(inv_freq, 4) ||
      !ns::aligned(q_out, 16))
    return -2;
  if (qkv_stride % 8 || qkv_stride < (Hq + 2ll * Hk) * D) return -2;
  const long long head = (long long)page_size * D;
  const ns::Bytes x = ns::rows_of(qkv, T, qkv_stride, (Hq + 2ll * Hk) * D, 2),
                  y = ns::bytes_of(q_out, 2 * (size_t)T * Hq * D), w = ns::bytes_of(bias, 2 * (Hq + 2ull * Hk) * D),
                  f = ns::bytes_of(inv_freq, 2 * (size_t)D);
  for (const ns::Bytes r : {x, y, w, f, ns::lens_of(a.s), ns::starts_of(a.s), ns::table_of(a.s)})
    if (!ns::pool_apart(a.p.k, a.p, Hk, head, r) || !ns::pool_apart(a.p.v, a.p, Hk, head, r)) return -2;
  if (!ns::apart(y, x) || !ns::apart(y, w) || !ns::apart(y, f)) return -2;
  if (!ns::pools_apart(a.p, Hk, head) || !ns::metadata_apart(a.s, y)) return -2;
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.bias = static_cast<const uint16_t*>(bias);
  a.inv_freq = static_cast<const float*>(inv_freq);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.qkv_stride = qkv_stride;
  a.Hq = Hq;
  a.Hk = Hk;
  a.D = D;
  const long long H = Hq + 2ll * Hk;
  if (T * H * (D / 16) >= (1ll << 38)) return -2;
  const auto st = static_cast<hipStream_t>(stream);
  if (T * H * (D / 16) <= ns::kSmall)
    ns::launch_append<1>(a, st);
  else
    ns::launch_append<6>(a, st);
  return static_cast<int>(hipGetLastError());
}
