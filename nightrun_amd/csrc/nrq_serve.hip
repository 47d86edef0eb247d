// C ABI of the serving operators (declared in include/nrq_serve.h): argument
// checks, then one or two kernel launches on the caller's stream.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "../../include/nrq.h"
#include "../../include/nrq_serve.h"
#include "nrq_launch.h"
#include "nrq_rows.h"
#include "nrq_serve_launch.h"

namespace {

static_assert(nrq::kF32 == NRQ_F32 && nrq::kF16 == NRQ_F16 && nrq::kBF16 == NRQ_BF16, "type ids");

int fail(int code, const char* name, const char* fmt, ...) {
  char buf[400], msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  snprintf(msg, sizeof msg, "%s: %s", name, buf);
  nrq::set_last_error(msg);
  return code;
}

// The library's device is the current one and the stream's.
int device_check(const char* name, void* stream) {
  const int dev = nrq::init_device();
  if (dev < 0) return fail(NRQ_ERR_NOT_INIT, name, "nrq_init was not called");
  int cur = -1;
  if (hipGetDevice(&cur) != hipSuccess) return fail(NRQ_ERR_DEVICE, name, "no current device");
  if (cur != dev)
    return fail(NRQ_ERR_ARG, name, "the current device is %d, the library was initialised on %d", cur, dev);
  int sdev = dev;
  if (stream && (hipStreamGetDevice((hipStream_t)stream, &sdev) != hipSuccess || sdev != dev))
    return fail(NRQ_ERR_ARG, name, "the stream is not on the library's device");
  return NRQ_OK;
}

int launched(const char* name, hipError_t e) {
  return e == hipSuccess ? NRQ_OK : fail(NRQ_ERR_DEVICE, name, "launch failed: %s", hipGetErrorString(e));
}

size_t bytes_of(int dtype) { return dtype == NRQ_F32 ? 4 : dtype == NRQ_F16 || dtype == NRQ_BF16 ? 2 : 0; }

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int kv_check(const char* name, const nrq_paged_kv* kv, const nrq_page_table* table, nrq::PagedKv* okv,
             nrq::PageTable* ot) {
  if (!kv) return fail(NRQ_ERR_ARG, name, "null cache");
  if (kv->dtype != NRQ_F16 && kv->dtype != NRQ_BF16) return fail(NRQ_ERR_ARG, name, "cache of unknown type %d", kv->dtype);
  if (kv->n_pages < 0 || kv->page_size < 1 || kv->n_kv_heads < 1 || kv->head_dim < 1)
    return fail(NRQ_ERR_SHAPE, name, "cache of %d pages of %d positions, %d heads of %d", kv->n_pages, kv->page_size,
                kv->n_kv_heads, kv->head_dim);
  if (kv->n_pages && (!kv->k || !kv->v)) return fail(NRQ_ERR_ARG, name, "null cache");
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(NRQ_ERR_ARG, name, "cache not 16-byte aligned");
  if (kv->page_stride < 0 || kv->head_stride < 0 || kv->pos_stride < 0 || kv->page_stride % 8 || kv->head_stride % 8 ||
      kv->pos_stride % 8)
    return fail(NRQ_ERR_ARG, name, "cache strides are not multiples of 8");
  // places count 8 elements in 32 bits, the last is no place; within a page there is no more than a page
  const double last = ((double)(kv->n_pages ? kv->n_pages - 1 : 0) * (double)kv->page_stride +
                       (double)(kv->page_size - 1) * (double)kv->pos_stride) / 8;
  if (last >= 4294967295.0 || kv->page_stride / 8 > 0xffffffffll || kv->pos_stride / 8 > 0xffffffffll)
    return fail(NRQ_ERR_UNSUPPORTED, name, "cache of more than 2^35 elements in a pool");
  *okv = nrq::PagedKv{(uint16_t*)kv->k, (uint16_t*)kv->v, kv->head_stride, (uint32_t)(kv->page_stride / 8),
                      (uint32_t)(kv->pos_stride / 8), kv->n_pages, kv->page_size, kv->n_kv_heads, kv->head_dim,
                      kv->dtype};
  if (!table) return NRQ_OK;
  if (table->seqs < 0 || table->width < 0) return fail(NRQ_ERR_SHAPE, name, "table of %d by %d", table->seqs, table->width);
  if (table->seqs && table->width && !table->pages) return fail(NRQ_ERR_ARG, name, "null table");
  if (!aligned(table->pages, 4)) return fail(NRQ_ERR_ARG, name, "table not aligned");
  *ot = nrq::PageTable{table->pages, table->stride, table->seqs, table->width};
  return NRQ_OK;
}

// Rows written must not overlap: sorted by their strides, each dimension steps over all of the ones inside it.
struct Dim {
  int64_t stride;
  size_t n;
};
bool apart(size_t row, std::initializer_list<Dim> dims) {
  Dim d[3];
  int count = 0;
  for (const Dim& x : dims) {
    if (x.n < 2) continue;
    int i = count++;
    for (; i > 0 && d[i - 1].stride > x.stride; i--) d[i] = d[i - 1];
    d[i] = x;
  }
  double extent = (double)row;  // of what lies inside; the strides may be anything
  for (int i = 0; i < count; i++) {
    if ((double)d[i].stride < extent) return false;
    extent += (double)d[i].stride * (double)(d[i].n - 1);
  }
  return true;
}

int rope_check(const char* name, const nrq::RopeLaunch& L, size_t tokens, size_t heads, size_t hd, size_t nf,
               int style) {
  if (!bytes_of(L.dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", L.dtype);
  if (style != NRQ_ROPE_ADJACENT && style != NRQ_ROPE_NEOX) return fail(NRQ_ERR_ARG, name, "unknown style %d", style);
  if (nf < 1 || hd > 1024 || nf > hd / 2)
    return fail(NRQ_ERR_SHAPE, name, "%zu frequencies for heads of %zu (at most half of them, at most 1024)", nf, hd);
  if (tokens > INT_MAX || heads > (size_t)1 << 20 || heads * hd > (size_t)1 << 20)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu tokens of %zu heads of %zu", tokens, heads, hd);
  if (!L.y || !L.x || !L.pos || !L.freqs) return fail(NRQ_ERR_ARG, name, "null pointer");
  const size_t e = bytes_of(L.dtype);
  if (!aligned(L.y, e) || !aligned(L.x, e) || !aligned(L.pos, 4) || !aligned(L.freqs, 4))
    return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  if (!apart(hd, {{L.yt, tokens}, {L.yh, heads}})) return fail(NRQ_ERR_ARG, name, "output rows overlap");
  if (L.y == L.x && (L.yt != L.xt || L.yh != L.xh))
    return fail(NRQ_ERR_ARG, name, "in place, but with other strides");
  return NRQ_OK;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

int workspace_check(const char* name, const void* p, size_t have, size_t need) {
  if (have < need) return fail(NRQ_ERR_ARG, name, "workspace of %zu bytes, %zu are needed", have, need);
  if (need && !p) return fail(NRQ_ERR_ARG, name, "null workspace");
  if (!aligned(p, 16)) return fail(NRQ_ERR_ARG, name, "workspace not 16-byte aligned");
  return NRQ_OK;
}

bool paged_hd(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

int mx_check(const char* name, size_t rows, size_t cols) {
  if (cols % 32) return fail(NRQ_ERR_SHAPE, name, "%zu columns are not a multiple of 32", cols);
  // both are rounded up to tiles in 32 bits
  if (rows > INT_MAX - 1024 || cols > INT_MAX - 1024) return fail(NRQ_ERR_UNSUPPORTED, name, "dimension exceeds 2^31");
  return NRQ_OK;
}

int mx_quant_check(const char* name, size_t rows, size_t cols) {
  int rc = mx_check(name, rows, cols);
  if (!rc && !nrq::mx_quantize_fits(rows, cols))
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu rows of %zu columns: more than 2^36 values", rows, cols);
  return rc;
}

size_t matmul_bytes(size_t rows, size_t cols, size_t batch) {
  return nrq::mx_matmul_workspace((int)rows, (int)cols, (int)batch);
}

// The activation in MXFP4 and what the product needs; few values the product's workgroups quantize for themselves.
size_t linear_own(size_t cols, size_t batch) { return up16(batch * (cols / 2)) + up16(batch * (cols / 32)); }
size_t linear_bytes(size_t rows, size_t cols, size_t batch) {
  if (nrq::mx_linear_fits((int)rows, (int)cols, (int)batch)) return 0;
  return linear_own(cols, batch) + matmul_bytes(rows, cols, batch);
}

int mx_matmul(const char* name, void* y, int dtype, int64_t ldy, const void* w, const void* ws, const void* x,
              const void* xs, size_t rows, size_t cols, size_t batch, void* workspace, void* stream) {
  nrq::MxMatmul L{y,         dtype,      ldy,        (const uint8_t*)w, (const uint8_t*)ws, (const uint8_t*)x, (const uint8_t*)xs,
                  (int)rows, (int)cols, (int)batch, (hipStream_t)stream, workspace};
  return launched(name, nrq::launch_mx_matmul(L));
}

int mx_product_check(const char* name, const void* y, int dtype, int64_t ldy, const void* w, const void* ws,
                     size_t rows, size_t cols, size_t batch) {
  int rc = mx_check(name, rows, cols);
  if (rc) return rc;
  if (!bytes_of(dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", dtype);
  if (batch > (size_t)1 << 20) return fail(NRQ_ERR_UNSUPPORTED, name, "batch of %zu (at most 2^20)", batch);
  if (!nrq::mx_matmul_fits((int)rows, (int)cols, (int)batch))
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu rows by %zu tokens: too many for a launch", rows, batch);
  if (!y || (cols && (!w || !ws))) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(y, bytes_of(dtype)) || !aligned(w, 16)) return fail(NRQ_ERR_ARG, name, "pointer not aligned");
  if (batch > 1 && ldy < (int64_t)rows) return fail(NRQ_ERR_ARG, name, "output rows overlap");
  return NRQ_OK;
}

// What a call of the MXFP4 functions writes shares no byte with what it reads or with another output: workgroups
// read while others write. Asked last, where the memory is known to be the device's.
nrq::Rows strided(const void* p, size_t n, int64_t stride, size_t cols, int dtype) {
  return nrq::Rows{p, n, stride, cols, (int)bytes_of(dtype)};
}
nrq::Rows packed(const void* q, size_t rows, size_t cols) { return nrq::Rows{q, 1, 0, rows * (cols / 2)}; }
nrq::Rows packed_scales(const void* s, size_t rows, size_t cols) { return nrq::Rows{s, 1, 0, rows * (cols / 32)}; }
int apart_check(const char* name, std::initializer_list<nrq::Rows> out, std::initializer_list<nrq::Rows> in) {
  for (const nrq::Rows* o = out.begin(); o != out.end(); o++) {
    for (const nrq::Rows& i : in)
      if (nrq::rows_meet(*o, i)) return fail(NRQ_ERR_ARG, name, "output and input overlap");
    for (const nrq::Rows* p = o + 1; p != out.end(); p++)
      if (nrq::rows_meet(*o, *p)) return fail(NRQ_ERR_ARG, name, "outputs overlap");
  }
  return NRQ_OK;
}

int mx_workspace(const char* name, size_t rows, size_t cols, size_t batch, size_t* bytes,
                 size_t (*need)(size_t, size_t, size_t)) {
  if (!bytes) return fail(NRQ_ERR_ARG, name, "null pointer");
  int rc = mx_check(name, rows, cols);
  if (rc) return rc;
  if (batch > (size_t)1 << 20) return fail(NRQ_ERR_UNSUPPORTED, name, "batch of %zu (at most 2^20)", batch);
  *bytes = need(rows, cols, batch);
  return NRQ_OK;
}

}  // namespace

extern "C" {

int nrq_dev_rope(void* y, const void* x, int dtype, size_t tokens, size_t heads, size_t head_dim,
                 const int64_t strides[4], const int32_t* pos, const float* freqs, size_t n_freqs, int style,
                 float scale, void* stream) {
  static const char* name = "nrq_dev_rope";
  int rc;
  if (tokens == 0 || heads == 0) return device_check(name, stream);
  if (!strides) return fail(NRQ_ERR_ARG, name, "null pointer");
  nrq::RopeLaunch L{};
  L.y = y, L.x = x, L.dtype = dtype, L.pos = pos, L.freqs = freqs;
  L.xt = strides[0], L.xh = strides[1], L.yt = strides[2], L.yh = strides[3];
  if ((rc = rope_check(name, L, tokens, heads, head_dim, n_freqs, style))) return rc;
  L.tokens = (int)tokens, L.heads = (int)heads, L.hd = (int)head_dim, L.nf = (int)n_freqs;
  L.neox = style == NRQ_ROPE_NEOX, L.scale = scale, L.stream = (hipStream_t)stream;
  if ((rc = device_check(name, stream))) return rc;
  return launched(name, nrq::launch_rope(L));
}

int nrq_dev_rope_append(void* y, const void* q, const void* k, const void* v, int dtype, size_t tokens, size_t heads,
                        const int64_t strides[8], const int32_t* pos, const int32_t* seq, const float* freqs,
                        size_t n_freqs, int style, float scale, const nrq_paged_kv* kv, const nrq_page_table* table,
                        void* stream) {
  static const char* name = "nrq_dev_rope_append";
  int rc;
  nrq::RopeLaunch L{};
  if (!table) return fail(NRQ_ERR_ARG, name, "null table");
  if ((rc = kv_check(name, kv, table, &L.kv, &L.table))) return rc;
  if (heads == 0) return fail(NRQ_ERR_SHAPE, name, "no heads");
  if (tokens == 0) return device_check(name, stream);
  if (!strides || !k || !v || !seq) return fail(NRQ_ERR_ARG, name, "null pointer");
  L.y = y, L.x = q, L.k = k, L.v = v, L.dtype = dtype, L.pos = pos, L.seq = seq, L.freqs = freqs;
  L.xt = strides[0], L.xh = strides[1], L.kt = strides[2], L.kh = strides[3];
  L.vt = strides[4], L.vh = strides[5], L.yt = strides[6], L.yh = strides[7];
  const size_t hd = (size_t)kv->head_dim;
  if ((rc = rope_check(name, L, tokens, heads, hd, n_freqs, style))) return rc;
  if ((size_t)kv->n_kv_heads * hd > (size_t)1 << 20) return fail(NRQ_ERR_UNSUPPORTED, name, "%d KV heads", kv->n_kv_heads);
  if (!apart(hd, {{kv->page_stride, (size_t)kv->n_pages}, {kv->head_stride, (size_t)kv->n_kv_heads}, {kv->pos_stride, (size_t)kv->page_size}}))
    return fail(NRQ_ERR_ARG, name, "the cache's positions overlap");
  if (!aligned(k, bytes_of(dtype)) || !aligned(v, bytes_of(dtype)) || !aligned(seq, 4))
    return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  L.tokens = (int)tokens, L.heads = (int)heads, L.hd = (int)hd, L.nf = (int)n_freqs;
  L.neox = style == NRQ_ROPE_NEOX, L.scale = scale, L.stream = (hipStream_t)stream;
  if ((rc = device_check(name, stream))) return rc;
  return launched(name, nrq::launch_rope(L));
}

int nrq_paged_attention_workspace(size_t seqs, size_t n_new, size_t heads, const nrq_paged_kv* kv, size_t* bytes) {
  static const char* name = "nrq_paged_attention_workspace";
  if (!bytes || !kv) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (kv->n_kv_heads < 1 || heads < 1 || heads % kv->n_kv_heads)
    return fail(NRQ_ERR_SHAPE, name, "%zu heads over %d KV heads", heads, kv->n_kv_heads);
  if (!paged_hd(kv->head_dim)) return fail(NRQ_ERR_UNSUPPORTED, name, "heads of %d", kv->head_dim);
  *bytes = nrq::paged_attn_workspace(seqs, n_new, heads, kv->n_kv_heads, kv->head_dim);
  return NRQ_OK;
}

int nrq_dev_paged_attention(void* out, const void* q, int dtype, size_t n_new, size_t heads, const int64_t strides[6],
                            const nrq_paged_kv* kv, const nrq_page_table* table, const int32_t* lens,
                            const int32_t* counts, float scale, int32_t window, float* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_paged_attention";
  int rc;
  nrq::PagedAttnLaunch L{};
  if (!table) return fail(NRQ_ERR_ARG, name, "null table");
  if ((rc = kv_check(name, kv, table, &L.kv, &L.table))) return rc;
  if (!bytes_of(dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", dtype);
  if (window < 0) return fail(NRQ_ERR_ARG, name, "window of %d", window);
  if (!paged_hd(kv->head_dim))
    return fail(NRQ_ERR_UNSUPPORTED, name, "heads of %d: 32, 64, 96, 128 or 256", kv->head_dim);
  if (heads < 1 || heads % kv->n_kv_heads)
    return fail(NRQ_ERR_SHAPE, name, "%zu heads over %d KV heads", heads, kv->n_kv_heads);
  if (table->seqs == 0 || n_new == 0) return device_check(name, stream);
  if (heads > 65536 || n_new > 65536 || n_new * heads > (size_t)1 << 20 ||
      n_new * heads * (size_t)table->seqs > (size_t)1 << 30)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%d sequences of %zu rows of %zu heads", table->seqs, n_new, heads);
  if (!strides || !out || !q || !lens) return fail(NRQ_ERR_ARG, name, "null pointer");
  const int64_t held = (int64_t)table->width * kv->page_size;  // positions of a sequence at most
  if (held > (int64_t)1 << 30) return fail(NRQ_ERR_UNSUPPORTED, name, "%lld positions of a sequence (at most 2^30)", (long long)held);
  if ((double)table->seqs * (double)(n_new * heads) * ((double)held / 128 + 1) >= 2147483647.0)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%d sequences of %d pages of %d: too much work for a call", table->seqs,
                table->width, kv->page_size);
  // the join takes a workgroup of 256 threads for each unit, and a grid has fewer than 2^32 of them
  if (nrq::paged_attn_units((size_t)table->seqs, n_new, heads, kv->n_kv_heads, kv->head_dim) >= (size_t)1 << 24 &&
      held > nrq::kPagedTile)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%d sequences of %zu rows of %zu heads: too much work for a call", table->seqs,
                n_new, heads);
  const size_t e = bytes_of(dtype);
  if (!aligned(out, e) || !aligned(q, e) || !aligned(lens, 4) || !aligned(counts, 4) || !aligned(lse, 4))
    return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  const size_t hd = (size_t)kv->head_dim;
  if (!apart(hd, {{strides[3], (size_t)table->seqs}, {strides[4], n_new}, {strides[5], heads}}))
    return fail(NRQ_ERR_ARG, name, "output rows overlap");
  if ((rc = workspace_check(name, workspace, workspace_bytes,
                            nrq::paged_attn_workspace((size_t)table->seqs, n_new, heads, kv->n_kv_heads, kv->head_dim))))
    return rc;
  L.out = out, L.q = q, L.dtype = dtype, L.n_new = (int)n_new, L.heads = (int)heads;
  L.qb = strides[0], L.qt = strides[1], L.qh = strides[2], L.ob = strides[3], L.ot = strides[4], L.oh = strides[5];
  // a window that no sequence outgrows is none (and position - window stays within 32 bits)
  L.lens = lens, L.counts = counts, L.scale = scale, L.window = window < held ? window : 0, L.lse = lse;
  L.workspace = workspace, L.stream = (hipStream_t)stream;
  if ((rc = device_check(name, stream))) return rc;
  return launched(name, nrq::launch_paged_attn(L));
}

int nrq_verify_workspace(size_t seqs, size_t vocab, size_t* bytes) {
  if (!bytes) return fail(NRQ_ERR_ARG, "nrq_verify_workspace", "null pointer");
  *bytes = nrq::verify_workspace(seqs, vocab);
  return NRQ_OK;
}

int nrq_dev_verify_drafts(int32_t* tokens, int32_t* accepted, const float* target, const float* draft,
                          const int64_t strides[4], const int32_t* drafted, const float* uniforms,
                          const int32_t* counts, size_t seqs, size_t n_new, size_t vocab, void* workspace,
                          size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_verify_drafts";
  int rc;
  if (n_new > 64) return fail(NRQ_ERR_UNSUPPORTED, name, "%zu drafted tokens (at most 64)", n_new);
  if (vocab < 1) return fail(NRQ_ERR_SHAPE, name, "empty vocabulary");
  if (vocab > (size_t)1 << 30 || seqs > (size_t)1 << 24)
    return fail(NRQ_ERR_UNSUPPORTED, name, "%zu sequences, vocabulary of %zu", seqs, vocab);
  if (seqs == 0) return device_check(name, stream);
  if (!strides || !tokens || !accepted || !target || !uniforms || (n_new && !drafted))
    return fail(NRQ_ERR_ARG, name, "null pointer");
  const void* words[] = {tokens, accepted, target, draft, drafted, uniforms, counts};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(NRQ_ERR_ARG, name, "pointer not aligned to its type");
  if ((rc = workspace_check(name, workspace, workspace_bytes, nrq::verify_workspace(seqs, vocab)))) return rc;
  nrq::VerifyLaunch L{tokens,     accepted,   target, draft,  strides[0], strides[1], strides[2], strides[3],
                      drafted,    uniforms,   counts, (int)seqs, (int)n_new, (int)vocab, workspace,  (hipStream_t)stream};
  if ((rc = device_check(name, stream))) return rc;
  return launched(name, nrq::launch_verify(L));
}

int nrq_dev_quantize_mxfp4(const void* src, int dtype, size_t rows, size_t cols, int64_t src_stride, void* q,
                           void* scales, void* stream) {
  static const char* name = "nrq_dev_quantize_mxfp4";
  int rc;
  if ((rc = mx_quant_check(name, rows, cols))) return rc;
  if (!bytes_of(dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", dtype);
  if (rows == 0 || cols == 0) return device_check(name, stream);
  if (!src || !q || !scales) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(src, bytes_of(dtype)) || !aligned(q, 16)) return fail(NRQ_ERR_ARG, name, "pointer not aligned");
  if ((rc = device_check(name, stream))) return rc;
  if ((rc = apart_check(name, {packed(q, rows, cols), packed_scales(scales, rows, cols)},
                        {strided(src, rows, src_stride, cols, dtype)})))
    return rc;
  return launched(name, nrq::launch_mx_quantize(src, dtype, rows, cols, src_stride, q, scales, (hipStream_t)stream));
}

int nrq_dev_dequantize_mxfp4(const void* q, const void* scales, size_t rows, size_t cols, void* dst, int dtype,
                             int64_t dst_stride, void* stream) {
  static const char* name = "nrq_dev_dequantize_mxfp4";
  int rc;
  if ((rc = mx_quant_check(name, rows, cols))) return rc;
  if (!bytes_of(dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", dtype);
  if (rows == 0 || cols == 0) return device_check(name, stream);
  if (!dst || !q || !scales) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(dst, bytes_of(dtype)) || !aligned(q, 16)) return fail(NRQ_ERR_ARG, name, "pointer not aligned");
  if (rows > 1 && dst_stride < (int64_t)cols) return fail(NRQ_ERR_ARG, name, "output rows overlap");
  if ((rc = device_check(name, stream))) return rc;
  if ((rc = apart_check(name, {strided(dst, rows, dst_stride, cols, dtype)},
                        {packed(q, rows, cols), packed_scales(scales, rows, cols)})))
    return rc;
  return launched(name, nrq::launch_mx_dequantize(q, scales, rows, cols, dst, dtype, dst_stride, (hipStream_t)stream));
}

int nrq_matmul_mxfp4_workspace(size_t rows, size_t cols, size_t batch, size_t* bytes) {
  return mx_workspace("nrq_matmul_mxfp4_workspace", rows, cols, batch, bytes, matmul_bytes);
}

int nrq_dev_matmul_mxfp4(void* y, int dtype, int64_t y_stride, const void* w, const void* w_scales, const void* x,
                         const void* x_scales, size_t rows, size_t cols, size_t batch, void* workspace,
                         size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_matmul_mxfp4";
  int rc;
  if (rows == 0 || batch == 0) return device_check(name, stream);
  if ((rc = mx_product_check(name, y, dtype, y_stride, w, w_scales, rows, cols, batch))) return rc;
  if (cols && (!x || !x_scales)) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(x, 16)) return fail(NRQ_ERR_ARG, name, "pointer not aligned");
  if ((rc = workspace_check(name, workspace, workspace_bytes, matmul_bytes(rows, cols, batch)))) return rc;
  if ((rc = device_check(name, stream))) return rc;
  if ((rc = apart_check(name, {strided(y, batch, y_stride, rows, dtype)},
                        {packed(w, rows, cols), packed_scales(w_scales, rows, cols), packed(x, batch, cols),
                         packed_scales(x_scales, batch, cols)})))
    return rc;
  return mx_matmul(name, y, dtype, y_stride, w, w_scales, x, x_scales, rows, cols, batch, workspace, stream);
}

int nrq_linear_mxfp4_workspace(size_t rows, size_t cols, size_t batch, size_t* bytes) {
  return mx_workspace("nrq_linear_mxfp4_workspace", rows, cols, batch, bytes, linear_bytes);
}

int nrq_dev_linear_mxfp4(void* y, int dtype, int64_t y_stride, const void* w, const void* w_scales, const void* x,
                         int x_dtype, int64_t x_stride, size_t rows, size_t cols, size_t batch, void* workspace,
                         size_t workspace_bytes, void* stream) {
  static const char* name = "nrq_dev_linear_mxfp4";
  int rc;
  if (rows == 0 || batch == 0) return device_check(name, stream);
  if ((rc = mx_product_check(name, y, dtype, y_stride, w, w_scales, rows, cols, batch))) return rc;
  if ((rc = mx_quant_check(name, batch, cols))) return rc;
  if (!bytes_of(x_dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", x_dtype);
  if (cols && !x) return fail(NRQ_ERR_ARG, name, "null pointer");
  if (!aligned(x, bytes_of(x_dtype))) return fail(NRQ_ERR_ARG, name, "pointer not aligned");
  if ((rc = workspace_check(name, workspace, workspace_bytes, linear_bytes(rows, cols, batch)))) return rc;
  if ((rc = device_check(name, stream))) return rc;
  if ((rc = apart_check(name, {strided(y, batch, y_stride, rows, dtype)},
                        {packed(w, rows, cols), packed_scales(w_scales, rows, cols),
                         strided(x, batch, x_stride, cols, x_dtype)})))
    return rc;
  if (cols && nrq::mx_linear_fits((int)rows, (int)cols, (int)batch)) {
    nrq::MxMatmul L{y,         dtype,      y_stride,   (const uint8_t*)w, (const uint8_t*)w_scales, nullptr, nullptr,
                    (int)rows, (int)cols, (int)batch, (hipStream_t)stream, nullptr};
    return launched(name, nrq::launch_mx_linear(L, x, x_dtype, x_stride));
  }
  uint8_t* xs = (uint8_t*)workspace + up16(batch * (cols / 2));
  if (cols && (rc = launched(name, nrq::launch_mx_quantize(x, x_dtype, batch, cols, x_stride, workspace, xs, (hipStream_t)stream))))
    return rc;
  return mx_matmul(name, y, dtype, y_stride, w, w_scales, workspace, xs, rows, cols, batch,
                   (uint8_t*)workspace + linear_own(cols, batch), stream);
}

}  // extern "C"
