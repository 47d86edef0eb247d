// C ABI of the operators for trees of drafts (declared in include/nrq_tree.h): argument
// checks, then one or two kernel launches on the caller's stream.
#include "../../include/nrq_tree.h"

#include "nrq_extent.h"
#include "nrq_serve_check.h"
#include "nrq_tree_launch.h"

namespace {

using nrq::Extent;
using nrq::Range;
using nrq::range_of;

Extent whole(const void* p, size_t n, int size) { return Extent{p, p ? n : 0, size, {}}; }

// Refuses outputs that share memory with one another or with inputs; those that are not there (nullptr) share none.
// Ranges that do not meet, as a rule, are told apart without more.
int apart_from(const char* name, std::initializer_list<Extent> out, std::initializer_list<Extent> in) {
  Range r[16];
  const Extent* e[16];
  size_t n = 0;
  const size_t outs = out.size();
  for (const auto* list : {&out, &in})
    for (const Extent& x : *list) {
      e[n] = &x;
      r[n++] = x.first ? range_of(x) : Range{1, 0};
    }
  for (size_t i = 0; i < outs; i++)
    for (size_t j = i + 1; j < n; j++)
      if (nrq::extents_meet(*e[i], r[i], *e[j], r[j]))
        return fail(NRQ_ERR_ARG, name, "an output shares memory with an input or another output");
  return NRQ_OK;
}

Extent heads_of(const void* p, int dtype, size_t tokens, int64_t ts, size_t heads, int64_t hs, size_t hd) {
  return Extent{p, hd, (int)bytes_of(dtype), {{ts, tokens}, {hs, heads}}};
}

Extent table_of(const nrq_page_table& t) {
  return Extent{t.pages, (size_t)t.width, 4, {{t.stride, (size_t)t.seqs}}};
}

Extent pool_of(const void* p, const nrq_paged_kv& kv) {
  return Extent{p, (size_t)kv.head_dim, 2,
                {{kv.page_stride, (size_t)kv.n_pages}, {kv.head_stride, (size_t)kv.n_kv_heads}, {kv.pos_stride, (size_t)kv.page_size}}};
}

int norm_check(const char* name, float eps, const float* wq, const float* wk) {
  if (!(eps >= 0.0f) || eps > 3e38f) return fail(NRQ_ERR_ARG, name, "eps of %g", (double)eps);
  if (!aligned(wq, 4) || !aligned(wk, 4)) return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  return NRQ_OK;
}

}  // namespace

extern "C" {

int nrq_dev_norm_rope(void* y, const void* x, int dtype, size_t tokens, size_t heads, size_t head_dim,
                      const int64_t strides[4], const float* weight, float eps, const int32_t* pos,
                      const float* freqs, size_t n_freqs, int style, float scale, void* stream) {
  static const char* name = "nrq_dev_norm_rope";
  int rc;
  if (tokens == 0 || heads == 0) return device_check(name, stream);
  if (!strides) return fail(NRQ_ERR_ARG, name, "null pointer");
  nrq::NormRopeLaunch N{};
  nrq::RopeLaunch& L = N.r;
  L.y = y, L.x = x, L.dtype = dtype, L.pos = pos, L.freqs = freqs;
  L.xt = strides[0], L.xh = strides[1], L.yt = strides[2], L.yh = strides[3];
  if ((rc = rope_check(name, L, tokens, heads, head_dim, n_freqs, style))) return rc;
  if ((rc = norm_check(name, eps, weight, nullptr))) return rc;
  L.tokens = (int)tokens, L.heads = (int)heads, L.hd = (int)head_dim, L.nf = (int)n_freqs;
  L.neox = style == NRQ_ROPE_NEOX, L.scale = scale, L.stream = (hipStream_t)stream;
  N.norm = true, N.wq = weight, N.eps = eps;
  if ((rc = device_check(name, stream))) return rc;
  // in place the input is left out
  if ((rc = apart_from(name, {heads_of(y, dtype, tokens, L.yt, heads, L.yh, head_dim)},
                       {heads_of(y != x ? x : nullptr, dtype, tokens, L.xt, heads, L.xh, head_dim),
                        whole(weight, head_dim, 4), whole(pos, tokens, 4), whole(freqs, n_freqs, 4)})))
    return rc;
  return launched(name, nrq::launch_norm_rope(N));
}

int nrq_dev_norm_rope_append(void* y, const void* q, const void* k, const void* v, int dtype, size_t tokens,
                             size_t heads, const int64_t strides[8], int norm, const float* q_weight,
                             const float* k_weight, float eps, const int32_t* pos, const int32_t* seq,
                             const int32_t* at, const float* freqs, size_t n_freqs, int style, float scale,
                             const nrq_paged_kv* kv, const nrq_page_table* table, void* stream) {
  static const char* name = "nrq_dev_norm_rope_append";
  int rc;
  nrq::NormRopeLaunch N{};
  nrq::RopeLaunch& L = N.r;
  if (!table) return fail(NRQ_ERR_ARG, name, "null table");
  if ((rc = kv_check(name, kv, table, &L.kv, &L.table))) return rc;
  if (heads == 0) return fail(NRQ_ERR_SHAPE, name, "no heads");
  if (tokens == 0) return device_check(name, stream);
  if (!strides || !k || !v || !seq) return fail(NRQ_ERR_ARG, name, "null pointer");
  L.y = y, L.x = q, L.k = k, L.v = v, L.dtype = dtype, L.pos = pos, L.seq = seq, L.freqs = freqs;
  L.xt = strides[0], L.xh = strides[1], L.kt = strides[2], L.kh = strides[3];
  L.vt = strides[4], L.vh = strides[5], L.yt = strides[6], L.yh = strides[7];
  const size_t hd = (size_t)kv->head_dim, n_kv = (size_t)kv->n_kv_heads;
  if ((rc = rope_check(name, L, tokens, heads, hd, n_freqs, style))) return rc;
  if (n_kv * hd > (size_t)1 << 20) return fail(NRQ_ERR_UNSUPPORTED, name, "%d KV heads", kv->n_kv_heads);
  if (!apart(hd, {{kv->page_stride, (size_t)kv->n_pages}, {kv->head_stride, n_kv}, {kv->pos_stride, (size_t)kv->page_size}}))
    return fail(NRQ_ERR_ARG, name, "the cache's positions overlap");
  if (!aligned(k, bytes_of(dtype)) || !aligned(v, bytes_of(dtype)) || !aligned(seq, 4) || !aligned(at, 4))
    return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  if (norm && (rc = norm_check(name, eps, q_weight, k_weight))) return rc;
  L.tokens = (int)tokens, L.heads = (int)heads, L.hd = (int)hd, L.nf = (int)n_freqs;
  L.neox = style == NRQ_ROPE_NEOX, L.scale = scale, L.stream = (hipStream_t)stream;
  N.norm = norm != 0, N.wq = q_weight, N.wk = k_weight, N.eps = eps, N.at = at;
  if ((rc = device_check(name, stream))) return rc;
  const Extent qe = heads_of(q, dtype, tokens, L.xt, heads, L.xh, hd), ke = heads_of(k, dtype, tokens, L.kt, n_kv, L.kh, hd),
               ve = heads_of(v, dtype, tokens, L.vt, n_kv, L.vh, hd), ye = heads_of(y, dtype, tokens, L.yt, heads, L.yh, hd),
               ck = pool_of(kv->k, *kv), cv = pool_of(kv->v, *kv);
  const Extent at_ = whole(at, tokens, 4), wq = whole(norm ? q_weight : nullptr, hd, 4), wk = whole(norm ? k_weight : nullptr, hd, 4),
               pe = whole(pos, tokens, 4), se = whole(seq, tokens, 4), fe = whole(freqs, n_freqs, 4), te = table_of(*table);
  const Extent none{};  // in place the queries are left out
  if ((rc = apart_from(name, {ye}, {y != q ? qe : none, ck, cv, ke, ve, pe, se, at_, fe, wq, wk, te})) ||
      (rc = apart_from(name, {ck}, {y != q ? qe : none, ke, ve, pe, se, at_, fe, wq, wk, te})) ||
      (rc = apart_from(name, {cv}, {y != q ? qe : none, ke, ve, pe, se, at_, fe, wq, wk, te})))
    return rc;
  if (nrq::copies_meet(ck, kv->v)) return fail(NRQ_ERR_ARG, name, "the cache's keys share memory with its values");
  return launched(name, nrq::launch_norm_rope(N));
}

int nrq_tree_attention_workspace(size_t seqs, size_t n_new, size_t heads, const nrq_paged_kv* kv, size_t* bytes) {
  static const char* name = "nrq_tree_attention_workspace";
  if (!bytes || !kv) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (kv->n_kv_heads < 1 || heads < 1 || heads % kv->n_kv_heads)
    return fail(NRQ_ERR_SHAPE, name, "%zu heads over %d KV heads", heads, kv->n_kv_heads);
  if (!paged_hd(kv->head_dim)) return fail(NRQ_ERR_UNSUPPORTED, name, "heads of %d", kv->head_dim);
  if (n_new > nrq::kTreeMost) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu nodes (at most 64)", n_new);
  *bytes = nrq::tree_attn_workspace(seqs, n_new, heads, kv->n_kv_heads, kv->head_dim);
  return NRQ_OK;
}

int nrq_dev_tree_attention(void* out, const void* q, int dtype, size_t n_new, size_t heads, const int64_t strides[6],
                           const nrq_paged_kv* kv, const nrq_page_table* table, const int32_t* lens,
                           const int32_t* parents, const int32_t* counts, float scale, int32_t window, float* lse,
                           void* workspace, size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_tree_attention";
  int rc;
  nrq::PagedAttnLaunch L{};
  if (n_new > nrq::kTreeMost) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu nodes (at most 64)", n_new);
  if ((rc = attn_check(name, out, q, dtype, n_new, heads, strides, kv, table, lens, counts, scale, window, lse, &L))) return rc;
  if (!L.out) return device_check(name, stream);  // nothing to do
  if (!parents) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(parents, 4)) return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  if (nrq::tree_attn_line((size_t)table->seqs, n_new, heads, kv->n_kv_heads, (int64_t)table->width * kv->page_size) >= 2147483647.0)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%d sequences of %d pages of %d: too much work for a call", table->seqs,
                table->width, kv->page_size);
  const size_t need = nrq::tree_attn_workspace((size_t)table->seqs, n_new, heads, kv->n_kv_heads, kv->head_dim);
  if ((rc = workspace_check(name, workspace, workspace_bytes, need))) return rc;
  L.parents = parents, L.workspace = workspace, L.stream = (hipStream_t)stream;
  if ((rc = device_check(name, stream))) return rc;
  const size_t hd = (size_t)kv->head_dim, seqs = (size_t)table->seqs, e = bytes_of(dtype);
  if ((rc = apart_from(name,
                       {{out, hd, (int)e, {{L.ob, seqs}, {L.ot, n_new}, {L.oh, heads}}},
                        whole(workspace, need, 1),
                        whole(lse, seqs * n_new * heads, 4)},
                       {{q, hd, (int)e, {{L.qb, seqs}, {L.qt, n_new}, {L.qh, heads}}},
                        whole(lens, seqs, 4),
                        whole(parents, seqs * n_new, 4),
                        whole(counts, seqs, 4),
                        table_of(*table),
                        pool_of(kv->k, *kv),
                        pool_of(kv->v, *kv)})))
    return rc;
  return launched(name, nrq::launch_tree_attn(L));
}

int nrq_verify_tree_workspace(size_t seqs, size_t vocab, size_t* bytes) {
  if (!bytes) return fail(NRQ_ERR_ARG, "nrq_verify_tree_workspace", "null pointer");
  *bytes = nrq::verify_tree_workspace(seqs, vocab);
  return NRQ_OK;
}

int nrq_dev_verify_tree(int32_t* tokens, int32_t* path, int32_t* accepted, const float* target,
                        const int64_t strides[2], const int32_t* drafted, const int32_t* parents,
                        const float* uniforms, const int32_t* counts, size_t seqs, size_t n_new, size_t vocab,
                        void* workspace, size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_verify_tree";
  int rc;
  if (n_new > nrq::kTreeMost) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu nodes (at most 64)", n_new);
  if (n_new < 1) return fail(NRQ_ERR_SHAPE, name, "a tree without a root");
  if (vocab < 1) return fail(NRQ_ERR_SHAPE, name, "empty vocabulary");
  if (vocab > (size_t)1 << 30 || seqs > (size_t)1 << 24)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu sequences, vocabulary of %zu", seqs, vocab);
  if (seqs == 0) return device_check(name, stream);
  if (!strides || !tokens || !path || !accepted || !target || !drafted || !parents || !uniforms)
    return fail(NRQ_ERR_ARG, name, "null pointer");
  const void* words[] = {tokens, path, accepted, target, drafted, parents, uniforms, counts};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  const size_t need = nrq::verify_tree_workspace(seqs, vocab), all = seqs * n_new;
  if ((rc = workspace_check(name, workspace, workspace_bytes, need))) return rc;
  nrq::VerifyLaunch L{tokens,   accepted, target, nullptr,    strides[0], strides[1], 0,         0,
                      drafted,  uniforms, counts, (int)seqs, (int)n_new, (int)vocab, workspace, (hipStream_t)stream,
                      parents,  path};
  if ((rc = device_check(name, stream))) return rc;
  if ((rc = apart_from(name, {whole(tokens, all, 4), whole(path, all, 4), whole(accepted, seqs, 4), whole(workspace, need, 1)},
                       {{target, vocab, 4, {{strides[0], seqs}, {strides[1], n_new}}},
                        whole(drafted, all, 4), whole(parents, all, 4), whole(uniforms, all, 4), whole(counts, seqs, 4)})))
    return rc;
  return launched(name, nrq::launch_verify_tree(L));
}

int nrq_dev_keep_path(int32_t* new_lens, size_t layers, int64_t layer_stride, const nrq_paged_kv* kv,
                      const nrq_page_table* table, const int32_t* lens, const int32_t* path, const int32_t* counts,
                      size_t n_new, void* stream) {
  static const char* name = "nrq_dev_keep_path";
  int rc;
  nrq::KeepLaunch L{};
  if (!table) return fail(NRQ_ERR_ARG, name, "null table");
  if ((rc = kv_check(name, kv, table, &L.kv, &L.table))) return rc;
  if (n_new > nrq::kTreeMost) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu nodes (at most 64)", n_new);
  const size_t n_kv = (size_t)kv->n_kv_heads, hd = (size_t)kv->head_dim, seqs = (size_t)table->seqs;
  if (n_kv * hd > (size_t)1 << 20) return fail(NRQ_ERR_UNSUPPORTED, name, "%d KV heads of %d", kv->n_kv_heads, kv->head_dim);
  if (seqs > (size_t)1 << 30) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu sequences (at most 2^30)", seqs);
  if (layers > (size_t)1 << 12) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu layers (at most 4096)", layers);
  // a thread has eight dimensions (the last of a head fewer) of keys or values, and the threads of a sequence are an int
  const double threads = 2.0 * (double)layers * (double)n_kv * (double)((hd + 7) / 8);
  if ((double)layers * (double)n_kv * (double)hd > 1073741824.0 || threads > (double)(INT_MAX - 255))
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu layers of %d KV heads of %d", layers, kv->n_kv_heads, kv->head_dim);
  const int64_t held = (int64_t)table->width * kv->page_size;  // positions of a sequence at most
  if (held > (int64_t)1 << 30) return fail(NRQ_ERR_UNSUPPORTED, name, "%lld positions of a sequence (at most 2^30)", (long long)held);
  if (seqs == 0) return device_check(name, stream);
  if (!new_lens || !lens || (n_new && !path)) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(new_lens, 4) || !aligned(lens, 4) || !aligned(path, 4) || !aligned(counts, 4))
    return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  if (layers > 1 && (layer_stride < 0 || layer_stride % 8)) return fail(NRQ_ERR_ARG, name, "layer stride is not a multiple of 8");
  if (!apart(hd, {{layer_stride, layers},
                  {kv->page_stride, (size_t)kv->n_pages},
                  {kv->head_stride, n_kv},
                  {kv->pos_stride, (size_t)kv->page_size}}))
    return fail(NRQ_ERR_ARG, name, "the caches' positions overlap");
  L.new_lens = new_lens, L.layers = (int)layers, L.layer_stride = layers > 1 ? layer_stride : 0;
  L.lens = lens, L.path = path, L.counts = counts, L.n_new = (int)n_new, L.stream = (hipStream_t)stream;
  if ((rc = device_check(name, stream))) return rc;
  const Extent le = whole(lens, seqs, 4), pe = whole(path, seqs * n_new, 4), ce = whole(counts, seqs, 4), te = table_of(*table);
  Extent ck = pool_of(kv->k, *kv), cv = pool_of(kv->v, *kv);
  ck.d[3] = cv.d[3] = {layer_stride, layers};
  if ((rc = apart_from(name, {whole(new_lens, seqs, 4)}, {ck, cv, le, pe, ce, te})) ||
      (rc = apart_from(name, {ck}, {le, pe, ce, te})) || (rc = apart_from(name, {cv}, {le, pe, ce, te})))
    return rc;
  if (nrq::copies_meet(ck, kv->v)) return fail(NRQ_ERR_ARG, name, "the cache's keys share memory with its values");
  return launched(name, nrq::launch_keep(L));
}

}  // extern "C"
