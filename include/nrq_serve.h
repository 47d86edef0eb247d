/*
 * libnrq — operators of a serving step, C ABI (second header of the library; include/nrq.h has the rest).
 *
 * Rotary positions with the append to a paged key-value cache, attention of the
 * new tokens over that cache, verification of drafted tokens, and the
 * microscaled 4-bit format MXFP4 with its product. No counterpart in the
 * reference, which runs one sequence over one contiguous cache.
 *
 * All pointers are device pointers on the device given to nrq_init, which has to
 * be the current one. Calls are asynchronous on `stream` (a hipStream_t of that
 * device; NULL = the null stream), allocate nothing, keep nothing between calls
 * and may be captured into a HIP graph. Two calls may run at the same time if
 * they write different memory (outputs, workspaces, cache positions). Strides
 * are in elements; the last dimension of every tensor is contiguous. Integers
 * that live on the device (lengths, positions, table entries, drafted tokens)
 * cannot be refused: what each function does with those out of range is said
 * there, and none reads or writes outside the tensors. Refused are, before
 * anything is launched: a current device or a stream of another device than
 * nrq_init's (NRQ_ERR_ARG), and sizes past what a call can take (NRQ_ERR_UNSUPPORTED).
 */
#ifndef NRQ_SERVE_H
#define NRQ_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types beside NRQ_F32 (0): IEEE binary16 and bfloat16 */
#define NRQ_F16 16
#define NRQ_BF16 17

/* A paged key-value cache: two pools of `n_pages` pages of `page_size`
 * positions, one for keys and one for values, of the same strides. The value of
 * position t of a sequence, KV head h, dimension d is at
 *   v[page * page_stride + h * head_stride + (t % page_size) * pos_stride + d]
 * with page = table[sequence][t / page_size]. Strides are multiples of 8, the
 * pools 16-byte aligned, a pool at most 2^35 elements. Any page size from 1. */
typedef struct {
  void *k, *v;
  int64_t page_stride, head_stride, pos_stride;
  int32_t n_pages, page_size, n_kv_heads, head_dim;
  int32_t dtype; /* NRQ_F16 or NRQ_BF16 */
} nrq_paged_kv;

/* Page numbers of `seqs` sequences, `width` of them for each, rows `stride`
 * apart. An entry outside [0, n_pages) is no page. */
typedef struct {
  const int32_t *pages;
  int64_t stride;
  int32_t seqs, width;
} nrq_page_table;

/* Rotary positions: with a = pos[t] * freqs[i] (the product and its reduction
 * in 64 bits), pair i of each head of token t becomes
 *   y0 = scale * (x0 cos a - x1 sin a),  y1 = scale * (x0 sin a + x1 cos a).
 * Pair i is (2i, 2i + 1) (NRQ_ROPE_ADJACENT) or (i, i + n_freqs)
 * (NRQ_ROPE_NEOX) of the head's first 2 n_freqs dimensions; the others are
 * copied. Context scaling goes into freqs and scale. x and y are
 * [tokens][heads][head_dim] of `dtype` (NRQ_F32, NRQ_F16, NRQ_BF16), strides =
 * {x token, x head, y token, y head}; y may be x (then with the same strides), but
 * may not overlap it otherwise. Any int32 position. 2 n_freqs <= head_dim <= 1024. */
int nrq_dev_rope(void *y, const void *x, int dtype, size_t tokens, size_t heads, size_t head_dim,
                 const int64_t strides[4], const int32_t *pos, const float *freqs, size_t n_freqs, int style,
                 float scale, void *stream);

/* The same rotation of q [tokens][heads][head_dim] into y and of k
 * [tokens][n_kv_heads][head_dim] into the cache, with v as it is, rounded to the
 * cache's type (to nearest, ties to even): token t goes to position pos[t] of
 * sequence seq[t]. strides = {q token, q head, k token, k head, v token, v head,
 * y token, y head}; y may be q. A token whose seq is outside [0, table.seqs) or
 * whose pos is negative is padding: its row of y stays as it was and nothing is
 * appended. A token whose position is behind the table, or on no page, is
 * rotated but not appended. At least one head of q. Where two tokens name the same position the cache
 * gets values of one or the other. */
int nrq_dev_rope_append(void *y, const void *q, const void *k, const void *v, int dtype, size_t tokens, size_t heads,
                        const int64_t strides[8], const int32_t *pos, const int32_t *seq, const float *freqs,
                        size_t n_freqs, int style, float scale, const nrq_paged_kv *kv, const nrq_page_table *table,
                        void *stream);

/* Attention of each sequence's last tokens over its cached positions. q and out
 * are [table.seqs][n_new][heads][head_dim] of `dtype` (NRQ_F32, NRQ_F16,
 * NRQ_BF16), strides = {q sequence, q token, q head, out sequence, out token, out
 * head}; heads is a multiple of the KV heads, query head h reads KV head h /
 * (heads / n_kv_heads). head_dim is 32, 64, 96, 128 or 256; a table holds at
 * most 2^30 positions of a sequence; n_new heads is at most 2^20.
 *   lens[b]: positions of sequence b, its new tokens' among them (their keys and
 *     values are in the cache already); below 0 is 0, more than the table holds
 *     is what it holds.
 *   counts[b] (or counts NULL: n_new): new tokens of sequence b, at its first
 *     counts[b] rows, in [0, n_new] (clamped); the rows behind them are left as they were.
 * Row j is the token at position p = lens[b] - counts[b] + j and attends to
 * positions t <= p, with window > 0 only to t > p - window; positions on no page
 * are not attended to. out = sum_t softmax_t(scale q.k_t) v_t; a row that attends
 * to nothing gives zeros. What the cache holds at positions that a row does not
 * attend to, infinities and NaN too, does not reach it. lse (or NULL):
 * f32 [table.seqs][n_new][heads] contiguous, log sum_t exp(scale q.k_t), -inf for nothing.
 * out may not overlap q. Scores, softmax and sums are in 32 bits; in products with an f16 cache, queries of another type
 * and the weights of the softmax are within 2^-23 of their value, or 2^-37 of the largest. The results depend on how the work
 * is split, never on the order in which it runs: the same call gives the same
 * bits.
 * workspace: nrq_paged_attention_workspace bytes, 16-byte aligned, its contents
 * of no meaning before and after; calls that may overlap, and graphs whose
 * replays may, need one each. */
int nrq_paged_attention_workspace(size_t seqs, size_t n_new, size_t heads, const nrq_paged_kv *kv, size_t *bytes);
int nrq_dev_paged_attention(void *out, const void *q, int dtype, size_t n_new, size_t heads, const int64_t strides[6],
                            const nrq_paged_kv *kv, const nrq_page_table *table, const int32_t *lens,
                            const int32_t *counts, float scale, int32_t window, float *lse, void *workspace,
                            size_t workspace_bytes, void *stream);

/* Verification of drafted tokens by rejection: per sequence b, drafted token
 * d_i, i = 0 .. n - 1, is accepted while
 *   uniforms[b][i] * draft[b][i][d_i] < target[b][i][d_i]
 * (draft NULL: the drafts were certain, draft[b][i][d_i] = 1). At the first i
 * refused a token is drawn from max(target[b][i] - draft[b][i], 0) (draft NULL:
 * target[b][i] without d_i; if that is zero throughout: target[b][i]); with all
 * accepted it is drawn from target[b][n]. Drawn is the smallest v whose
 * cumulative sum through v is above uniforms[b][n] (below 0: 0) * the whole sum,
 * else the last v with any weight; -1 if none has. Products, differences and sums are in 64 bits.
 * target is f32 [seqs][n_new + 1][vocab], draft f32 [seqs][n_new][vocab],
 * strides = {target sequence, target row, draft sequence, draft row}; drafted
 * int32 [seqs][n_new], uniforms f32 [seqs][n_new + 1], both contiguous; n =
 * counts[b] clamped to [0, n_new] (counts NULL: n_new; the last uniform is
 * always uniforms[b][n_new]). A drafted token outside the vocabulary is refused (and
 * has no draft weight to leave out). NaN counts as no weight, and refuses a draft.
 * tokens int32 [seqs][n_new + 1]: the accepted, the drawn one, then -1;
 * accepted int32 [seqs]: how many drafts were. n_new <= 64.
 * workspace: nrq_verify_workspace bytes, 16-byte aligned, as for the attention. */
int nrq_verify_workspace(size_t seqs, size_t vocab, size_t *bytes);
int nrq_dev_verify_drafts(int32_t *tokens, int32_t *accepted, const float *target, const float *draft,
                          const int64_t strides[4], const int32_t *drafted, const float *uniforms,
                          const int32_t *counts, size_t seqs, size_t n_new, size_t vocab, void *workspace,
                          size_t workspace_bytes, void *stream);

/* MXFP4 (the OCP microscaling formats' 4-bit one): blocks of 32 values along a
 * row share a scale 2^(s - 127), s a byte; each value is 4 bits: sign and 0,
 * .5, 1, 1.5, 2, 3, 4 or 6, two to a byte, the first in the low bits. q is
 * [rows][cols / 2] bytes, scales [rows][cols / 32] bytes, contiguous, q 16-byte
 * aligned; cols a multiple of 32. Scales have to be readable from the 16-byte
 * boundary before their first byte to the one behind their last (true within any
 * HIP allocation). s - 127 = floor(log2(largest magnitude)) - 2,
 * at least -127 (also for zeros); values to the nearest of those (ties to the even
 * code), at most 6. A block with an infinity or a NaN is s = 255 (NaN
 * throughout) with zeros. Here and in the functions below an output that shares memory with
 * an input or another output is refused; columns of one matrix do not. */
int nrq_dev_quantize_mxfp4(const void *src, int dtype, size_t rows, size_t cols, int64_t src_stride, void *q,
                           void *scales, void *stream);
/* The values of such blocks, rounded to `dtype`; dst rows dst_stride apart. */
int nrq_dev_dequantize_mxfp4(const void *q, const void *scales, size_t rows, size_t cols, void *dst, int dtype,
                             int64_t dst_stride, void *stream);
/* y[b][r] = sum_c x[b][c] * w[r][c] with both in MXFP4, the products exact, sums in 32 bits,
 * y [batch][rows] of `dtype`, rows of y y_stride apart. workspace: nrq_matmul_mxfp4_workspace
 * bytes (0 for many sizes: then NULL will do), 16-byte aligned, as for the attention. */
int nrq_matmul_mxfp4_workspace(size_t rows, size_t cols, size_t batch, size_t *bytes);
int nrq_dev_matmul_mxfp4(void *y, int dtype, int64_t y_stride, const void *w, const void *w_scales, const void *x,
                         const void *x_scales, size_t rows, size_t cols, size_t batch, void *workspace,
                         size_t workspace_bytes, void *stream);
/* The same with the activation quantized on the way: x [batch][cols] of x_dtype,
 * rows x_stride apart; the result is that of nrq_dev_quantize_mxfp4 and
 * nrq_dev_matmul_mxfp4. workspace: nrq_linear_mxfp4_workspace bytes, 16-byte
 * aligned, as for the attention. */
int nrq_linear_mxfp4_workspace(size_t rows, size_t cols, size_t batch, size_t *bytes);
int nrq_dev_linear_mxfp4(void *y, int dtype, int64_t y_stride, const void *w, const void *w_scales, const void *x,
                         int x_dtype, int64_t x_stride, size_t rows, size_t cols, size_t batch, void *workspace,
                         size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NRQ_SERVE_H */
