/*
 * batch_ops.h -- entry points of libnanoserve_amd.so for a batch of sequences over one paged KV
 * cache, which nanoserve_amd/ops.py calls (Kernels.paged_append, paged_attention, their forms for a cache in 8
 * bits, paged_reserve, beam_select, paged_reorder, sample) and the public headers do not declare. Conventions of include/nanoserve_decode.h: caller-allocated device
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
 * The same over a cache in 8 bits. Pools of e4m3 codes (strides in bytes, multiples of 16), and beside them scales: one
 * byte e per 16 rows of a page and head, for 2^(e - 127), at k_scales + page * scale_page_stride + head *
 * scale_head_stride + row / 16, v_scales alike. A value is code times scale.
 *
 * ns_paged_append_fp8: y as ns_paged_append's, in fp32. For the new rows of a block of 16 positions of one sequence and
 * kv head, K and V apart, t their largest finite magnitude: e' = the least with t <= 448 * 2^e', held to [-110, 119]; where
 * the block has rows from before (its first new position is no multiple of 16) the larger of that and the scale
 * there (held to the same), and those rows' codes become e4m3(code * 2^(e - e')). Codes are e4m3(y / 2^e'), rounded to
 * nearest even, held to 448; NaN and infinities become NaN. D 64 or 128, T * Hk < 2^29; -2 also for scales over anything
 * else, or over pages (where neither the spans are apart nor the page strides the same).
 * Two sequences that append to one page leave one of the two values of each element and scale, which need not
 * belong together.
 *
 * ns_paged_attention_fp8: ns_paged_attention over the values. The query enters the first product as two e4m3
 * terms under a power of two per head: exact down to 2^-14 of the head's largest magnitude, within 2^-22 of it below,
 * held to 448 * 2^119; infinities in it become NaN. A scale byte of 255 counts as 254.
 */
int ns_paged_append_fp8(const void* qkv, long long qkv_stride, const void* bias, const void* inv_freq,
                        const int* q_start, const int* lens, const int* table, long long table_stride,
                        int width, void* k_pool, void* v_pool, long long page_stride,
                        long long head_stride, void* k_scales, void* v_scales,
                        long long scale_page_stride, long long scale_head_stride, int n_pages,
                        int page_size, void* q_out, int T, int B, int Hq, int Hk, int D, void* stream);
size_t ns_paged_attention_fp8_workspace(int T, int B, int Hq, int Hk, int D, int max_len, int ragged,
                                        int shared);
int ns_paged_attention_fp8(const void* q, long long q_stride, const void* k_pool, const void* v_pool,
                           long long page_stride, long long head_stride, const void* k_scales,
                           const void* v_scales, long long scale_page_stride, long long scale_head_stride,
                           int n_pages, int page_size, const int* table, long long table_stride, int width,
                           const int* lens, const int* q_start, void* out, void* work, size_t work_bytes,
                           int T, int B, int Hq, int Hk, int D, int shared, int window, int sinks,
                           float scale, void* stream);

/*
 * Table entries, first rows and slot map of a step, from its sequences' new lengths: sequence b has lens[b] positions
 * (held to 0 .. width * page_size) and gets add[b] more, or gives back -add[b] of them. In place:
 *   lens [B]       becomes max(lens + add, 0)
 *   table          entries ceil(old / page_size) .. ceil(new / page_size) - 1 of a sequence that grows are taken from
 *                  the stack, in the order of the sequences and entries, its top first. The entries of one that shrinks
 *                  from ceil(new / page_size) on go back to it (and stay in the table), the last one first: what one call
 *                  took and a later one gives back lies there as before. Pages given back count for the same call.
 *   free, n_free   the stack: pages free[0 .. n_free[0] - 1], the top last, room for `capacity`
 * Written: q_start [B + 1], the running sum of max(add, 0) from 0 on; slots [rows], of each new token in that order
 * page * page_size + row, -1 where the table's entry is below 0 and behind the last sequence's (rows -1: no slot map, slots
 * unused); shorts [1]: 0.
 * A call that does not go through as a whole changes nothing: q_start is all 0 (rows of no sequence, on which the operators
 * that are given it do nothing; without it they take every sequence's last position for its new one), slots are -1, and shorts is the number of pages that are missing, or -1 where a sequence would pass its
 * table row, more than `rows` tokens are new, or the stack would pass its capacity.
 * n_free below 0 counts as 0, past the capacity the call does not go through. Entries given back must not be in use by other
 * rows. -2 for sizes <= 0 (B >= 2^24, rows < -1, capacity < 0 or >= 2^31),
 * page_size % 16, width * page_size >= 2^30, table_stride < width, NULL or misaligned pointers (slots 8, others 4
 * bytes), and any two of the arrays over each other.
 */
int ns_paged_reserve(const int* add, int* lens, int* table, long long table_stride, int width, int* free_pages,
                     long long capacity, int* n_free, int* q_start, long long* slots, int rows, int* shorts,
                     int B, int page_size, void* stream);

/*
 * Bytes of workspace ns_beam_select uses for these sizes, 0 for sizes it rejects. Launches that may overlap in time need
 * workspaces of their own.
 */
size_t ns_beam_select_workspace(int R, int beams, int V, int n);

/*
 * The n best continuations of each of R requests with `beams` beams. logits: R * beams rows (request-major) row_stride apart of V
 * values (bf16, or fp32 with fp32 != 0); scores [R][beams], what a beam has so far. With l the logits
 *   c[i][v] = scores[i] + l[i][v] - log(sum over v of exp(l[i][v]))
 * out_scores, out_tokens, out_parents [R][n] are the n largest c with their v and i, falling; within a beam in the order of
 * the logits, equal ones by rising v, between beams in that of c in 64 bits, equal ones by rising i. The exponentials are 32
 * bits wide, which moves a beam's c as a whole by 2^-22 or so: beams whose c lie closer may come in either order. NaN logits and scores count as -inf, +inf as the largest fp32; a score of
 * -inf is a beam that does not count, a logit of -inf is never taken. Where fewer than n are left: -inf, -1, -1.
 * -2 for sizes <= 0, beams or n above 64, R * beams > 65535, V > 2^20, row_stride < V, NULL or misaligned pointers (logits 2
 * or 4 bytes, work 16, others 4), work_bytes too small, outputs and the workspace over an input or each other.
 */
int ns_beam_select(const void* logits, int fp32, long long row_stride, const float* scores, float* out_scores,
                   int* out_tokens, int* out_parents, void* work, size_t work_bytes, int R, int beams, int V, int n,
                   void* stream);

/*
 * The pages of R requests' beams after a selection: beam i of a request goes on from beam parents[i] (rows parent_stride apart;
 * one that is not 0 .. beams - 1 counts as i). table and lens are those of the R * beams sequences, request-major; the
 * beams of a request have the same length n. out [R * beams][width] receives, per beam, with w = n / page_size whole
 * pages: entries 0 .. w - 1 of its parent; where n % page_size is not 0 entry w of a page of its own, which holds
 * the parent's rows; behind that the beam's own entries. Of a parent's children the parent itself, or else the first one,
 * keeps the parent's page w; the k-th of the others gets page w of the k-th beam that no one goes on from, into which the
 * n % page_size rows of every layer and head are copied in both pools, and the scales of their blocks (k_scales and
 * v_scales NULL: a cache without). The last, partly filled pages of a request must be the beams' own. table is not changed,
 * so a repeated call gives the same; entries outside [0, n_pages) are moved and not copied from or to.
 * Whole pages that only beams had which no one goes on from are in no row of out: ns_paged_reorder_back gives them back, or else
 * the caller has to keep count of a request's pages.
 * Pools: + layer * layer_stride + page * page_stride + head * head_stride + row * row_bytes (bytes, multiples of 16); scales
 * alike, one byte per 16 rows. -2 for sizes <= 0, beams > 64, R * beams >= 2^24, page_size % 16, width * page_size
 * >= 2^30, page_size * row_bytes * Hk >= 2^31, strides by which layers, pages and heads overlap, NULL or misaligned pointers
 * (pools 16, int 4 bytes), pages over each other (as in ns_paged_append_fp8), out or an input within the pools' spans, out over an input.
 */
int ns_paged_reorder(const int* parents, long long parent_stride, const int* table, long long table_stride, int width,
                     const int* lens, int* out, void* k_pool, void* v_pool, long long layer_stride,
                     long long page_stride, long long head_stride, void* k_scales, void* v_scales,
                     long long scale_layer_stride, long long scale_page_stride, long long scale_head_stride, int layers,
                     int n_pages, int page_size, int row_bytes, int R, int beams, int Hk, void* stream);

/*
 * ns_paged_reorder, and the whole pages (of columns below w) that are in rows of beams which no one goes on from and in no row of
 * one from which someone does are pushed on the stack of ns_paged_reserve, each once: free[n_free[0]] on, the last one the
 * top, in the order of the requests, their columns and in a column the beams. Entries outside [0, n_pages) are no pages. A
 * repeated call pushes them again. n_free below 0 counts as 0; past the capacity nothing is pushed, and what would lie past it
 * is left out: the stack needs room for every page. Pages that rows of another request hold too must be in all of a request's
 * rows (a common prefix is). -2 also for n_free NULL, free NULL with a capacity, capacity < 0 or >= 2^31, either misaligned (4
 * bytes), and the two over each other or anything else.
 */
int ns_paged_reorder_back(const int* parents, long long parent_stride, const int* table, long long table_stride, int width,
                          const int* lens, int* out, void* k_pool, void* v_pool, long long layer_stride,
                          long long page_stride, long long head_stride, void* k_scales, void* v_scales,
                          long long scale_layer_stride, long long scale_page_stride, long long scale_head_stride, int layers,
                          int n_pages, int page_size, int row_bytes, int R, int beams, int Hk, int* free,
                          long long capacity, int* n_free, void* stream);

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
