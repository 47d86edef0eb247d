// Internal launch interface of the serving operators (nrq_serve.hip checks the
// arguments; the kernel files launch). The public interface is include/nrq_serve.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nrq {

enum { kF32 = 0, kF16 = 16, kBF16 = 17 };

struct PagedKv {
  uint16_t *k, *v;
  int64_t head_stride;
  uint32_t page_stride8, pos_stride8;  // in units of 8 elements
  int n_pages, page_size, n_kv, hd;
  int dtype;
};

struct PageTable {
  const int* pages;
  int64_t stride;
  int seqs, width;
};

struct RopeLaunch {
  void* y;
  const void *x, *k, *v;  // k, v: nullptr without the append
  int dtype;
  int tokens, heads, hd;
  int64_t xt, xh, yt, yh, kt, kh, vt, vh;
  const int *pos, *seq;
  const float* freqs;
  int nf;
  bool neox;
  float scale;
  PagedKv kv;
  PageTable table;
  hipStream_t stream;
};
hipError_t launch_rope(const RopeLaunch& L);

struct PagedAttnLaunch {
  void* out;
  const void* q;
  int dtype;
  int n_new, heads;
  int64_t qb, qt, qh, ob, ot, oh;
  PagedKv kv;
  PageTable table;
  const int *lens, *counts;
  float scale;
  int window;
  float* lse;
  void* workspace;
  hipStream_t stream;
  const int* parents = nullptr;  // [seqs][n_new]: the new tokens are a tree's nodes (launch_tree_attn)
};
constexpr int kPagedTile = 128;  // positions of a tile; where a sequence holds no more there is no join
size_t paged_attn_units(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd);
size_t paged_attn_workspace(size_t seqs, size_t n_new, size_t heads, int n_kv, int hd);
hipError_t launch_paged_attn(const PagedAttnLaunch& L);

struct VerifyLaunch {
  int *tokens, *accepted;
  const float *target, *draft;
  int64_t tb, tr, db, dr;
  const int* drafted;
  const float* uniforms;
  const int* counts;
  int seqs, n_new, vocab;
  void* workspace;
  hipStream_t stream;
  const int* parents = nullptr;  // [seqs][n_new]: the drafted tokens are a tree's nodes (launch_verify_tree)
  int* path = nullptr;
};
size_t verify_workspace(size_t seqs, size_t vocab);
hipError_t launch_verify(const VerifyLaunch& L);
size_t verify_tree_workspace(size_t seqs, size_t vocab);
hipError_t launch_verify_tree(const VerifyLaunch& L);

bool mx_quantize_fits(size_t rows, size_t cols);  // whether a grid holds the values
hipError_t launch_mx_quantize(const void* src, int dtype, size_t rows, size_t cols, int64_t stride, void* q, void* s,
                              hipStream_t stream);
hipError_t launch_mx_dequantize(const void* q, const void* s, size_t rows, size_t cols, void* dst, int dtype,
                                int64_t stride, hipStream_t stream);
struct MxMatmul {
  void* y;
  int dtype;
  int64_t ldy;
  const uint8_t *w, *ws, *x, *xs;
  int rows, cols, batch;
  hipStream_t stream;
  void* workspace;
};
bool mx_matmul_fits(int rows, int cols, int batch);  // whether a grid holds the tiles
bool mx_gemm_fits(int rows, int cols, int batch);
size_t mx_matmul_workspace(int rows, int cols, int batch);
size_t mx_gemm_workspace(int rows, int cols, int batch);
hipError_t launch_mx_matmul(const MxMatmul& L);
bool mx_linear_fits(int rows, int cols, int batch);  // whether launch_mx_linear takes the activation as it is
hipError_t launch_mx_linear(const MxMatmul& L, const void* x, int x_dtype, int64_t stride);
hipError_t launch_mx_gemm(const MxMatmul& L);  // many tokens (nrq_mx_gemm.hip)

}  // namespace nrq
