/*
 * batch_ops.h -- entry points of libnanoserve_amd.so for a batch of sequences over one paged KV
 * cache, which nanoserve_amd/ops.py calls (Kernels.paged_append, paged_attention, sample) and the
 * public headers do not declare. Conventions of include/nanoserve_decode.h: caller-allocated device
 * memory, bf16 tensors as void*, asynchronous on `stream`, no allocation, no host synchronisation,
 * capturable; 0 on success, -2 for rejected arguments (checked before any HIP call), else the
 * hipError_t. The reference serves one sequence at a time (python/nanoserve/qwen.py:113-177) and has
 * no counterpart of these.
 *
 * A batch is described by device int32 arrays:
 *   q_start [B + 1]  token rows q_start[b] .. q_start[b + 1] - 1 are sequence b's new tokens, ascending
 *                    and inside [0, T]; NULL: one token per sequence (T == B, row b)
 *   lens [B]         positions of sequence b including its new tokens, which are the last ones: new
 *                    token i of nn is at position lens[b] - nn + i. A length past the table counts as
 *                    width * page_size, one below zero as zero.
 *   table [B][width] (rows table_stride apart) page of positions page_size * j .. of sequence b
 * Pages: pool + page * page_stride + kv head * head_stride + row * D (strides in elements), page_size
 * rows of D values, page_size a multiple of 16; K and V pools alike. A table entry outside
 * [0, n_pages) is no page: nothing is stored there and its positions are left out of the attention.
 * Entries past a sequence's length are not read.
 */
#ifndef NANOSERVE_BATCH_OPS_H
#define NANOSERVE_BATCH_OPS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Bias + position rotation + append of every new token of the batch. qkv [T] rows qkv_stride apart of
 * (Hq + 2 Hk) D values (q, k, v heads). With x = qkv + bias (bias NULL: qkv) in fp32 and
 * a = position * inv_freq[i] (fp64 product, i < D / 2):
 *   y[i] = x[i] cos a - x[i + D/2] sin a,  y[i + D/2] = x[i + D/2] cos a + x[i] sin a
 * for q and k heads, y = x for v heads, rounded once to bf16. q heads go to q_out [T][Hq * D], k and v
 * heads to their position's row of the pools. Token rows of no sequence are left alone, tokens before
 * position 0 (more new tokens than positions) are rotated and not stored. Two sequences whose tables
 * name the same page for a row that both write leave one of the two values of each element there.
 * -2 for D % 16, D > 512, sizes <= 0, page_size % 16, strides that are not a multiple of 8 or shorter
 * than what they span, width * page_size >= 2^30, NULL or misaligned pointers (bf16 16, int 4 bytes),
 * q_start NULL with T != B; pools that share rows with each other, with q_out or with an input, and q_out over an input
 * (qkv counts from its first value to its last, what lies between its rows included).
 */
int ns_paged_append(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq,
                    const int* q_start, const int* lens, const int* table, long long table_stride,
                    int width, void* k_pool, void* v_pool, long long page_stride,
                    long long head_stride, int n_pages, int page_size, void* q_out, int T, int B,
                    int Hq, int Hk, int D, void* stream);

/*
 * Bytes of workspace ns_paged_attention uses for these sizes (max_len = width * page_size; ragged:
 * q_start is given), 0 for none or for sizes it rejects. Launches that may overlap in time need
 * workspaces of their own.
 */
size_t ns_paged_attention_workspace(int T, int B, int Hq, int Hk, int D, int max_len, int ragged,
                                    int shared);

/*
 * Grouped-query attention of the batch's new tokens over the pages (their own keys and values
 * included: append first). A token at position p of sequence b sees position j if j <= p and, with
 * window > 0, j > p - window or j < sinks. out [T][Hq * D] bf16 = softmax(scale q . K) V over what it
 * sees, zeros where that is nothing; token rows of no sequence are left alone. q: rows q_stride apart,
 * heads contiguous. Products of bf16 operands, softmax and all sums in fp32; probabilities enter the
 * second product as two bf16 terms (16 significant bits).
 * shared > 0: the caller states that positions 0 .. shared - 1, as far as a sequence has them, lie in the
 * same pages for every sequence; they are read through the row of the longest one, once for the batch.
 * A head's output is NaN for NaN in its query or in a key that it sees, for a score of +inf and for scores that are
 * all -inf. Keys and values (NaN and infinities among them) in positions that no token sees have no effect. A NaN
 * or infinite value that a token sees leaves that dimension of its output NaN or infinite (NaN also where the exact
 * result is infinite: the second term of a probability is zero or negative), and may do so to the tokens of the same
 * kv head in its launch tile that do not see it.
 * -2 for D other than 64 and 128, Hq % Hk, T * Hq >= 2^30, negative window, sinks or shared, scale not positive and
 * finite, and as ns_paged_append (the pools may be one and the same here); work_bytes too small; out and the workspace
 * over each other or over an input.
 */
int ns_paged_attention(const void* q, long long q_stride, const void* k_pool, const void* v_pool,
                       long long page_stride, long long head_stride, int n_pages, int page_size,
                       const int* table, long long table_stride, int width, const int* lens,
                       const int* q_start, void* out, void* work, size_t work_bytes, int T, int B,
                       int Hq, int Hk, int D, int shared, int window, int sinks, float scale,
                       void* stream);

/*
 * Bytes of workspace ns_sample uses for these sizes, 0 for none or for sizes it rejects. Launches that
 * may overlap in time need workspaces of their own.
 */
size_t ns_sample_workspace(int B, int V, int fp32);

/*
 * One token per row of logits [B] rows row_stride apart of V values (bf16, or fp32 with fp32 != 0),
 * from a given random number u [B] in [0, 1). Per row, with l the logits, T the temperature and
 * z_i = (l_i - max l) / T, w_i = exp(z_i):
 *   - order the tokens by falling logit, equal ones by rising index
 *   - keep the first top_k (all for top_k <= 0)
 *   - of those keep the shortest beginning whose weights reach top_p of their sum (all for
 *     top_p >= 1, at least one)
 *   - of those keep the ones with w_i >= min_p (min_p above 1 counts as 1)
 *   - out = the first token, by index, at which the running sum of the kept weights exceeds u times
 *     their whole sum
 * T <= 0: the first token of that order. NaN logits count as -inf, +inf as the largest fp32; -inf is never
 * drawn; out = -1 where nothing is left. u below 0 (or NaN) counts as 0, u from 1 on as the last kept token.
 * Settings per row: temps, top_ks, top_ps, min_ps [B] device arrays, each NULL for the scalar beside it.
 * Weights are held in units of 2^-42 of the largest in 64-bit integers and summed exactly, so the token
 * does not depend on the order of any sum.
 * -2 for B <= 0, B > 65535, V <= 0, V > 2^20, row_stride < V, NULL or misaligned pointers (logits 2 or 4
 * bytes, int and float 4, work 16), work_bytes too small, out over the logits (from the first row to the last),
 * the workspace over anything else.
 */
int ns_sample(const void* logits, int fp32, long long row_stride, const float* u, const float* temps,
              float temp, const int* top_ks, int top_k, const float* top_ps, float top_p,
              const float* min_ps, float min_p, int* out, void* work, size_t work_bytes, int B, int V,
              void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NANOSERVE_BATCH_OPS_H */
