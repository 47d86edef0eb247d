/*
 * libnrq — operators of a serving step whose drafted tokens form a tree, C ABI (third header of the library).
 *
 * Norms of queries and keys with the rotary positions in the same pass, attention of a
 * tree's nodes over a paged cache, acceptance of a path through the tree, and the move of that
 * path's keys and values to the places where they belong. What include/nrq_serve.h says of
 * pointers, streams, strides, devices, errors, overlapping calls and integers on the device holds here too.
 *
 * A tree of n nodes, at most 64: node 0 is its root, the last token known; parents[j] is the node that
 * node j follows, 0 <= parents[j] < j. A parent outside that range is none: such a node (the root is one)
 * has nothing above it in the tree. The nodes' keys and values are the last n of a sequence's cached
 * positions: node j is at base + j, base = lens[b] - n. Its rotary position is base plus the number of nodes above it.
 */
#ifndef NRQ_TREE_H
#define NRQ_TREE_H

#include "nrq_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

/* nrq_dev_rope of normed rows: each head's row x of head_dim values becomes
 *   x / sqrt(mean of x^2 + eps) * weight
 * before it is rotated, in 32 bits throughout and rounded once: a row whose squares add up to 2^128 or more becomes
 * zeros, and a square below 2^-150 is 0. weight is f32
 * [head_dim], the same for all heads (NULL: ones). eps >= 0; a row of zeros with eps 0 gives NaN. Arguments else as
 * for nrq_dev_rope; y may be x (then with the same strides), but shares no memory with it otherwise, and none with weight, pos or freqs. */
int nrq_dev_norm_rope(void *y, const void *x, int dtype, size_t tokens, size_t heads, size_t head_dim,
                      const int64_t strides[4], const float *weight, float eps, const int32_t *pos,
                      const float *freqs, size_t n_freqs, int style, float scale, void *stream);

/* nrq_dev_rope_append of normed rows: q with q_weight, k with k_weight (NULL: ones), v as it is. norm 0: q and k
 * as they are (weights and eps are not used). at (or NULL: pos) has the cache position of each token, where it
 * is not the rotary one; then pos may be any int32. A token whose seq is outside [0, table.seqs) or whose place at[t] is
 * negative is padding, one whose place is behind the table, or on no page, is rotated but not appended. y may be q (then with the
 * same strides); it shares no memory with q otherwise, nor with any other input, the cache none with either, and
 * its keys none with its values. */
int nrq_dev_norm_rope_append(void *y, const void *q, const void *k, const void *v, int dtype, size_t tokens,
                             size_t heads, const int64_t strides[8], int norm, const float *q_weight,
                             const float *k_weight, float eps, const int32_t *pos, const int32_t *seq,
                             const int32_t *at, const float *freqs, size_t n_freqs, int style, float scale,
                             const nrq_paged_kv *kv, const nrq_page_table *table, void *stream);

/* nrq_dev_paged_attention where the new tokens are the nodes of a tree: counts[b] of them (or counts NULL:
 * n_new <= 64), clamped to [0, n_new]; the rows behind them are left as they were. parents is int32
 * [table.seqs][n_new], contiguous. Row j attends to the positions before base, and at base and behind it to node j and the nodes above
 * it alone; with window > 0 only to what is less than `window` rotary positions before its own. Where lens[b] is less than the
 * nodes, those at negative positions are attended to by none. Arguments, empty rows, precision and workspace
 * (nrq_tree_attention_workspace) else as for nrq_dev_paged_attention; out and lse share no memory with the inputs or one
 * another. An infinity among the values that a row attends to is the row's output, however small its weight (where its score is
 * -infinity, a NaN). What an infinity or a NaN in the cache costs: rows of its KV head are done again one position after the other, so that a long
 * sequence takes a hundred times as long. How rows are shared out goes by the table's width, as the lengths are on the device: in a
 * table far wider than its sequences are long, short ones take up to a third longer. */
int nrq_tree_attention_workspace(size_t seqs, size_t n_new, size_t heads, const nrq_paged_kv *kv, size_t *bytes);
int nrq_dev_tree_attention(void *out, const void *q, int dtype, size_t n_new, size_t heads, const int64_t strides[6],
                           const nrq_paged_kv *kv, const nrq_page_table *table, const int32_t *lens,
                           const int32_t *parents, const int32_t *counts, float scale, int32_t window, float *lse,
                           void *workspace, size_t workspace_bytes, void *stream);

/* Acceptance of a path through a tree of drafts that were certain (the draft's best tokens). Row j of target, f32
 * [seqs][n_new][vocab], strides = {sequence, row}, has the probabilities of what follows node j. Per sequence, from the
 * root on: the children of the node reached are tried in order, child j with token x = drafted[b][j] accepted if
 *   target[b][node][x] > 0  and  uniforms[b][j] * left < target[b][node][x]
 * with left = 1 minus the probabilities of the node's children refused before, added up in their order; a token
 * that one of those had has none left. The accepted child is the next node reached. Where none is accepted, or there
 * is none, a token is drawn from target[b][node] without the tokens refused (if that is zero throughout: target[b][node]): the
 * smallest v whose cumulative sum through v is above uniforms[b][0] (below 0: 0) * the whole sum, else the last v with
 * any weight; -1 if none has. Products, differences and sums are in 64 bits. So the accepted tokens and the
 * drawn one are distributed as if each had been drawn from the target alone. drafted, parents int32 and uniforms f32 are
 * [seqs][n_new], contiguous (drafted[b][0] is not read); counts[b] (or counts NULL: n_new) is the number of nodes, clamped to
 * [0, n_new]. A token outside the vocabulary is refused and takes nothing away; NaN and what is below 0 count as no weight.
 * accepted int32 [seqs]: the number of drafts accepted, a. tokens int32 [seqs][n_new]: their tokens, the one drawn,
 * then -1. path int32 [seqs][n_new]: the nodes from the root on, a + 1 of them, then -1. A sequence without nodes
 * gives 0 and -1 throughout. n_new <= 64. The outputs share no memory with one another or the inputs.
 * workspace: nrq_verify_tree_workspace bytes, 16-byte aligned, as for the attention. */
int nrq_verify_tree_workspace(size_t seqs, size_t vocab, size_t *bytes);
int nrq_dev_verify_tree(int32_t *tokens, int32_t *path, int32_t *accepted, const float *target,
                        const int64_t strides[2], const int32_t *drafted, const int32_t *parents,
                        const float *uniforms, const int32_t *counts, size_t seqs, size_t n_new, size_t vocab,
                        void *workspace, size_t workspace_bytes, void *stream);

/* Moves the keys and values of an accepted path to where a sequence without the other nodes has them, in `layers`
 * caches that share one table: the pools of layer l begin l * layer_stride elements (a multiple of 8) behind kv->k and kv->v. With
 * n = counts[b] (or counts NULL: n_new) nodes, clamped to [0, n_new], and base = lens[b] - n (lens[b] below 0 is 0,
 * more than the table holds is what it holds), position base + i gets what position base + path[b][i] had, for
 * the leading entries of path[b] (int32 [table.seqs][n_new], contiguous) that grow and lie in [0, n): the first that does not
 * ends the path. new_lens[b] (int32 [table.seqs]) = base + the number of those, at least 0. A move from or to a
 * position that is negative or on no page is left out. What was behind the new length is of no meaning.
 * Where two sequences of a call have a page in common, neither may write to it. new_lens shares no memory with the
 * inputs or the caches, these none with the inputs, keys none with values. n_new <= 64, at most 2^30 sequences. A layer
 * has at most 2^20 values of a position (KV heads times head_dim, any head_dim), all layers, 4096 at most, have at most
 * 2^30, in at most 2^30 - 128 eights (the last of a head may be short). */
int nrq_dev_keep_path(int32_t *new_lens, size_t layers, int64_t layer_stride, const nrq_paged_kv *kv,
                      const nrq_page_table *table, const int32_t *lens, const int32_t *path, const int32_t *counts,
                      size_t n_new, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NRQ_TREE_H */
