// What the C entries of the serving operators check alike: errors, devices, caches, rows that overlap.
#pragma once

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "../../include/nrq.h"
#include "../../include/nrq_serve.h"
#include "nrq_extent.h"
#include "nrq_launch.h"
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
using nrq::Dim;
bool apart(size_t row, std::initializer_list<Dim> dims) {
  Dim d[4];
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

int workspace_check(const char* name, const void* p, size_t have, size_t need) {
  if (have < need) return fail(NRQ_ERR_ARG, name, "workspace of %zu bytes, %zu are needed", have, need);
  if (need && !p) return fail(NRQ_ERR_ARG, name, "null workspace");
  if (!aligned(p, 16)) return fail(NRQ_ERR_ARG, name, "workspace not 16-byte aligned");
  return NRQ_OK;
}

bool paged_hd(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// The arguments of an attention over a paged cache, as a launch without workspace and stream; out is left nullptr where there is nothing to do.
int attn_check(const char* name, void* out, const void* q, int dtype, size_t n_new, size_t heads, const int64_t strides[6],
               const nrq_paged_kv* kv, const nrq_page_table* table, const int32_t* lens, const int32_t* counts, float scale,
               int32_t window, float* lse, nrq::PagedAttnLaunch* launch) {
  int rc;
  nrq::PagedAttnLaunch& L = *launch;
  if (!table) return fail(NRQ_ERR_ARG, name, "null table");
  if ((rc = kv_check(name, kv, table, &L.kv, &L.table))) return rc;
  if (!bytes_of(dtype)) return fail(NRQ_ERR_ARG, name, "unknown type %d", dtype);
  if (window < 0) return fail(NRQ_ERR_ARG, name, "window of %d", window);
  if (!paged_hd(kv->head_dim))
    return fail(NRQ_ERR_UNSUPPORTED, name, "heads of %d: 32, 64, 96, 128 or 256", kv->head_dim);
  if (heads < 1 || heads % kv->n_kv_heads)
    return fail(NRQ_ERR_SHAPE, name, "%zu heads over %d KV heads", heads, kv->n_kv_heads);
  if (table->seqs == 0 || n_new == 0) return NRQ_OK;
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
  L.out = out, L.q = q, L.dtype = dtype, L.n_new = (int)n_new, L.heads = (int)heads;
  L.qb = strides[0], L.qt = strides[1], L.qh = strides[2], L.ob = strides[3], L.ot = strides[4], L.oh = strides[5];
  // a window that no sequence outgrows is none (and position - window stays within 32 bits)
  L.lens = lens, L.counts = counts, L.scale = scale, L.window = window < held ? window : 0, L.lse = lse;
  return NRQ_OK;
}

}  // namespace
