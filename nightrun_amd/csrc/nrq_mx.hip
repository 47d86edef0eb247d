// MXFP4 (include/nrq_serve.h): quantization, its inverse, and the product of
// two quantized matrices on the scaled matrix instructions.
//
// v_mfma_scale_f32_16x16x128 takes from lane l the 32 values of one block: row
// l % 16 of its operand, columns 32 (l / 16) .. + 31 of the step's 128, 16
// consecutive bytes of the row, and the block's scale byte. The product of two
// values has at most 4 significant bits, so the sums within a block are exact.
//
// All three are bound by memory where they are not by the launch: 9728 x 2560 of bf16 to 4 bits
// and back (113 MB) takes 22 us, 5.1 TB/s; one f32 token by 19456 x 2560 (26 MB of weights)
// 7.3 us, 3.6 TB/s, its quantization in the same launch.
#include "nrq_serve_launch.h"

namespace nrq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct alignas(16) Half16 {
  T v[16 / sizeof(T)];
};

// Eight values of a row: 16 bytes (wide 2: streamed past the caches) or, for unaligned rows, one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int wide, float* f) {
  constexpr int V = 16 / sizeof(T);
  if (wide == 2) {
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      const i32x4 x = __builtin_nontemporal_load((const i32x4*)(p + i));
      const Half16<T> a = *(const Half16<T>*)&x;
#pragma unroll
      for (int j = 0; j < V; j++) f[i + j] = (float)a.v[j];
    }
  } else if (wide) {
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      const Half16<T> a = *(const Half16<T>*)(p + i);
#pragma unroll
      for (int j = 0; j < V; j++) f[i + j] = (float)a.v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)p[i];
  }
}

// One block from four lanes of eight values each: the lane's 8 codes, and the scale.
__device__ __forceinline__ uint32_t mx_quantize8(float* f, uint32_t* scale) {
  uint32_t top = 0;  // magnitudes order like their bits; infinity and NaN on top
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  const bool bad = top >= 0x7f800000u;
  // floor(log2) is the exponent field, less the two binades up to 4; subnormal
  // and small blocks keep the smallest scale
  const int e = (int)(top >> 23) - 2;
  const uint32_t s = (uint32_t)max(e, 0);
  *scale = bad ? 255u : s;
  const float by = __uint_as_float(s ? s << 23 : 0x00400000u);
  uint32_t r = 0;
  if (!bad) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[0], f[1], by, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[2], f[3], by, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[4], f[5], by, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[6], f[7], by, 3);
  }
  return r;
}

constexpr int kMxOwn = 16384;  // values that a workgroup of four waves quantizes for itself
constexpr int kMxAhead = 2;  // accesses of a thread that are on their way together

// Eight values an access, four lanes a block: cols / 8 is a multiple of four and a workgroup
// starts at a multiple of four, so a block's lanes stay together. dense: rows without gaps.
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* src, int64_t stride, uint32_t cols8, int64_t items,
                                                          uint32_t* q, uint8_t* sc, int wide, int dense) {
  const int64_t i0 = (int64_t)blockIdx.x * (256 * kMxAhead) + threadIdx.x;
  float f[kMxAhead][8];
#pragma unroll
  for (int k = 0; k < kMxAhead; k++) {
    const int64_t i = min(i0 + 256 * k, items - 1);  // no load is conditional
    const int64_t row = dense ? 0 : i / cols8;
    load8(src + (dense ? i * 8 : row * stride + (i - row * cols8) * 8), wide, f[k]);
  }
#pragma unroll
  for (int k = 0; k < kMxAhead; k++) {
    const int64_t i = i0 + 256 * k;
    if (i >= items) break;
    uint32_t s;
    q[i] = mx_quantize8(f[k], &s);
    if ((threadIdx.x & 3) == 0) sc[i >> 2] = (uint8_t)s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* q, const uint8_t* sc, int64_t stride,
                                                            uint32_t cols8, int64_t items, T* dst, int wide, int dense) {
  const int64_t i0 = (int64_t)blockIdx.x * (256 * kMxAhead) + threadIdx.x;
  uint32_t w[kMxAhead], s[kMxAhead];
#pragma unroll
  for (int k = 0; k < kMxAhead; k++) {
    const int64_t i = min(i0 + 256 * k, items - 1);
    w[k] = q[i];
    s[k] = sc[i >> 2];
  }
#pragma unroll
  for (int k = 0; k < kMxAhead; k++) {
    const int64_t i = i0 + 256 * k;
    if (i >= items) break;
    const float by = __uint_as_float(s[k] == 255u ? 0x7fc00000u : (s[k] ? s[k] << 23 : 0x00400000u));
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      // code eem: 2^(ee - 1) (1 + m / 2), or m / 2
      const uint32_t n = (w[k] >> (4 * e)) & 15u, ee = (n >> 1) & 3u, m = n & 1u;
      const float mag = ee ? __uint_as_float(((ee + 126u) << 23) | (m << 22)) : 0.5f * m;
      f[e] = (n & 8u ? -mag : mag) * by;
    }
    const int64_t row = dense ? 0 : i / cols8;
    T* d = dst + (dense ? i * 8 : row * stride + (i - row * cols8) * 8);
    constexpr int V = 16 / sizeof(T);
    if (wide) {
#pragma unroll
      for (int e = 0; e < 8; e += V) {
        Half16<T> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.v[j] = (T)f[e + j];
        // streamed: 9728 x 2560 bf16 takes 11.6 us so, 17.7 with ordinary stores
        __builtin_nontemporal_store(*(i32x4*)&o, (i32x4*)(d + e));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) d[e] = (T)f[e];
    }
  }
}

// One lane's block: 16 bytes and its scale.
struct MxBlock {
  i32x4 q;
  int s;
};
__device__ __forceinline__ MxBlock mx_block(const uint8_t* q, const uint8_t* s) { return MxBlock{*(const i32x4*)q, (int)*s}; }

__device__ __forceinline__ f32x4 mx_mfma(const MxBlock& a, const MxBlock& b, f32x4 c) {
  const i32x8 x = {a.q.x, a.q.y, a.q.z, a.q.w, 0, 0, 0, 0}, y = {b.q.x, b.q.y, b.q.z, b.q.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, a.s, 0, b.s);
}

template <typename T>
__device__ __forceinline__ void put4(T* p, int64_t at, int n, f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i < n) p[at + i] = (T)v[i];
}

__device__ __forceinline__ void mx_store(void* y, int dtype, int64_t at, int n, f32x4 v) {
  if (dtype == kF32)
    put4((float*)y, at, n, v);
  else if (dtype == kF16)
    put4((_Float16*)y, at, n, v);
  else
    put4((__bf16*)y, at, n, v);
}

// Tiles of 16 rows of w by 16 NT tokens. A workgroup's W waves take every
// W-th step of 128 columns and add up in LDS; it goes from one row tile to another, the next
// weights on their way while these are multiplied. With X the activation is not in MXFP4
// yet but [batch][cols] of X: every workgroup quantizes it once into LDS, behind the loads of its
// first weights, which saves a launch (for a token or a few: see mx_linear_fits).
template <int NT, int U, int W, typename X>
__global__ __launch_bounds__(64 * W) void mx_matvec_kernel(MxMatmul L, int tiles, const X* act, int64_t stride, int wide) {
  constexpr bool kOwn = !__is_same(X, void);
  __shared__ f32x4 part[2][W][NT][64];
  extern __shared__ __align__(16) uint8_t own[];  // with X: [batch][cols / 2], then [batch][cols / 32]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, steps = (blocks + 3) / 4;
  MxBlock a[U];
  auto load = [&](int tile, int s0) {
    const int row = tile * 16 + i;
    const int64_t r = (int64_t)min(row, L.rows - 1) * blocks;
#pragma unroll
    for (int u = 0; u < U; u++) {
      // blocks behind the last read the last again, no load is conditional; they are cleared when used
      const int64_t b = r + min(4 * (s0 + W * u) + g, blocks - 1);
      a[u] = mx_block(L.w + b * 16, L.ws + b);
    }
  };
  const uint8_t *xq = L.x, *xs = L.xs;
  if constexpr (kOwn) {
    // the first two accesses of each thread are asked for before the weights: loads come back in order
    uint8_t* oq = own;
    uint8_t* os = own + (size_t)L.batch * blocks * 16;
    const int cols8 = L.cols / 8, items = L.batch * cols8;
    auto value = [&](int k, float* f) {
      const int t = L.batch == 1 ? 0 : k / cols8;
      load8(act + t * stride + (k - t * cols8) * 8, wide, f);
    };
    auto put = [&](int k, float* f) {
      uint32_t s;
      ((uint32_t*)oq)[k] = mx_quantize8(f, &s);
      if ((k & 3) == 0) os[k >> 2] = (uint8_t)s;
    };
    float f[2][8];
    const int t = threadIdx.x;
    value(min(t, items - 1), f[0]);
    value(min(t + 64 * W, items - 1), f[1]);
    load(blockIdx.x, w);
    if (t < items) put(t, f[0]);
    if (t + 64 * W < items) put(t + 64 * W, f[1]);
    for (int k = t + 128 * W; k < items; k += 64 * W) {
      value(k, f[0]);
      put(k, f[0]);
    }
    __syncthreads();
    xq = oq, xs = os;
  } else if (blocks) {
    load(blockIdx.x, w);
  }
  int round = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, round++) {
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f32x4{0, 0, 0, 0};
    for (int s0 = w; s0 < steps; s0 += W * U) {
      MxBlock now[U];
#pragma unroll
      for (int u = 0; u < U; u++) now[u] = a[u];
      if (s0 + W * U < steps)
        load(tile, s0 + W * U);
      else if (tile + (int)gridDim.x < tiles)
        load(tile + gridDim.x, w);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int b = 4 * (s0 + W * u) + g;
        const bool none = b >= blocks;
        if (none) now[u] = MxBlock{{0, 0, 0, 0}, 127};
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const int tok = min((int)(blockIdx.y * NT + t) * 16 + i, L.batch - 1);  // tokens behind the last are not stored
          const int64_t at = (int64_t)tok * blocks + min(b, blocks - 1);
          MxBlock x = mx_block(xq + at * 16, xs + at);
          if (none) x.s = 127;
          acc[t] = mx_mfma(now[u], x, acc[t]);
        }
      }
    }
    // one barrier a tile: the wave that adds a tile up has done so before the barrier of the next, after
    // which its place is written again
    auto& p = part[round & 1];
#pragma unroll
    for (int t = 0; t < NT; t++) p[w][t][lane] = acc[t];
    __syncthreads();
    if (w != (round & (W - 1))) continue;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      f32x4 y = p[0][t][lane];
#pragma unroll
      for (int k = 1; k < W; k++) y += p[k][t][lane];
      const int tok = (blockIdx.y * NT + t) * 16 + i, r = tile * 16 + 4 * g;
      if (tok < L.batch && r < L.rows) mx_store(L.y, L.dtype, tok * L.ldy + r, L.rows - r, y);
    }
  }
}

// Workgroups for `tiles` row tiles: all of them up to 2048, else few enough that each has as many (65536 x 4096
// by one and three tokens: 35.8 and 41.4 us, 36.6 and 47.3 with one tile a workgroup; 128256 x 2048 by one 35.6 and 35.3, by
// three 38.5 and 40.9; 19456 x 2560 by one is all of them: 7.8, with 768 8.9).
inline unsigned mx_matvec_grid(int tiles) {
  const int rounds = (tiles + 2047) / 2048;
  return (unsigned)((tiles + rounds - 1) / rounds);
}

// Eight waves a workgroup, where there are no more workgroups than CUs and rows long enough for them, else four: 2048 x
// 8192 by one and four tokens takes 6.2 and 10.3 us with eight, 7.3 and 12.1 with four, 2560 x 9728 by one 6.8 and 7.7.
// Steps of a wave on their way together (U): four or five, whichever divides its steps with less rest (2048 columns
// are four steps a wave, 2560 five: 128256 x 2048 by one takes 35.7 us with four and 41.9 with five, 19456 x 2560 10.1 and 7.3).
template <int W, typename X>
void matvec_w(const MxMatmul& L, size_t lds, const X* x, int64_t stride, int wide) {
  const int tiles = (L.rows + 15) / 16, steps = (L.cols + 128 * W - 1) / (128 * W);
  const dim3 grid(mx_matvec_grid(tiles));
  if ((steps + 3) / 4 * 4 < (steps + 4) / 5 * 5)
    hipLaunchKernelGGL((mx_matvec_kernel<1, 4, W, X>), grid, dim3(64 * W), lds, L.stream, L, tiles, x, stride, wide);
  else
    hipLaunchKernelGGL((mx_matvec_kernel<1, 5, W, X>), grid, dim3(64 * W), lds, L.stream, L, tiles, x, stride, wide);
}

inline bool mx_wide(int rows, int cols) { return rows <= 16 * 256 && cols >= 4096; }

template <typename X>
void matvec_t(const MxMatmul& L, size_t lds, const X* x, int64_t stride, int wide) {
  if (mx_wide(L.rows, L.cols))
    matvec_w<8>(L, lds, x, stride, wide);
  else
    matvec_w<4>(L, lds, x, stride, wide);
}

template <typename T>
bool wide_rows(const void* p, int64_t stride) {
  return ((uintptr_t)p & 15) == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
}

inline unsigned mx_grid(int64_t items) { return (unsigned)((items + 256 * kMxAhead - 1) / (256 * kMxAhead)); }

template <typename T>
void quantize_t(const void* src, size_t rows, size_t cols, int64_t stride, void* q, void* s, hipStream_t st) {
  const int64_t items = (int64_t)rows * (cols / 8);
  // more than the L2s hold is streamed: 9728 x 2560 bf16 and back takes 22.0 us so, 23.9 through them; less stays in
  // them (2048 x 2048 f32 before its product: 73.4 us streamed, 72.4 not)
  const bool big = items * 8 * (int64_t)sizeof(T) > 32 << 20;
  hipLaunchKernelGGL((mx_quantize_kernel<T>), dim3(mx_grid(items)), dim3(256), 0, st, (const T*)src, stride,
                     (uint32_t)(cols / 8), items, (uint32_t*)q, (uint8_t*)s, wide_rows<T>(src, stride) ? (big ? 2 : 1) : 0,
                     stride == (int64_t)cols || rows == 1);
}

template <typename T>
void dequantize_t(const void* q, const void* s, size_t rows, size_t cols, void* dst, int64_t stride, hipStream_t st) {
  const int64_t items = (int64_t)rows * (cols / 8);
  hipLaunchKernelGGL((mx_dequantize_kernel<T>), dim3(mx_grid(items)), dim3(256), 0, st, (const uint32_t*)q,
                     (const uint8_t*)s, stride, (uint32_t)(cols / 8), items, (T*)dst, wide_rows<T>(dst, stride) ? 1 : 0,
                     stride == (int64_t)cols || rows == 1);
}

template <typename X>
void linear_t(const MxMatmul& L, const void* x, int64_t stride) {
  const size_t lds = (size_t)L.batch * (L.cols / 2 + L.cols / 32);
  matvec_t<X>(L, lds, (const X*)x, stride, wide_rows<X>(x, stride) ? 1 : 0);
}

}  // namespace

// Grids of fewer than 2^24 workgroups of 256 threads: a launch takes fewer than 2^32 threads.
bool mx_quantize_fits(size_t rows, size_t cols) { return (double)rows * (double)(cols / 8) <= 256.0 * kMxAhead * 16777215.0; }

hipError_t launch_mx_quantize(const void* src, int dtype, size_t rows, size_t cols, int64_t stride, void* q, void* s,
                              hipStream_t st) {
  if (dtype == kF32)
    quantize_t<float>(src, rows, cols, stride, q, s, st);
  else if (dtype == kF16)
    quantize_t<_Float16>(src, rows, cols, stride, q, s, st);
  else
    quantize_t<__bf16>(src, rows, cols, stride, q, s, st);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const void* q, const void* s, size_t rows, size_t cols, void* dst, int dtype,
                                int64_t stride, hipStream_t st) {
  if (dtype == kF32)
    dequantize_t<float>(q, s, rows, cols, dst, stride, st);
  else if (dtype == kF16)
    dequantize_t<_Float16>(q, s, rows, cols, dst, stride, st);
  else
    dequantize_t<__bf16>(q, s, rows, cols, dst, stride, st);
  return hipGetLastError();
}

// The tiles of 128 x 128: from 65 tokens on, or where there are many rows (64 x 9728 x 2560: 14.8 us on them, 20.5
// not; 4 x 128256 x 2048: 35.8 and 40.9, but 1 x 32768 x 2560: 14.8 and 10.9) or columns, which workgroups share
// out (17 x 2560 x 9728: 14.4 and 21.3, 64: 15.5 and 34; but 17 x 2048 x 2560: 13.5 and 9.3). Their scales come in
// pairs at least.
static bool mx_wants_gemm(int rows, int cols, int batch) {
  return cols >= 64 && (batch > 64 || (batch > 16 && (rows >= 8192 || cols >= 4096)) || (batch > 3 && rows >= 32768));
}

// A token or a few are quantized by every workgroup of the product, up to 16384 values, twice as many by one of eight
// waves: 9728 x 2560 by one, four, eight tokens takes 6.3, 7.7, 10.1 us so and 9.7, 10.2, 10.1 in two launches, 4096 x 4096
// by eight and twelve 7.3, 9.3 and 9.8, 10.0, 2048 x 8192 by four and eight 10.0, 13.9 and 10.4, 10.7.
bool mx_linear_fits(int rows, int cols, int batch) {
  return batch <= 16 && (int64_t)cols * batch <= (mx_wide(rows, cols) ? 2 * kMxOwn : kMxOwn) && !mx_wants_gemm(rows, cols, batch);
}

hipError_t launch_mx_linear(const MxMatmul& L, const void* x, int x_dtype, int64_t stride) {
  if (x_dtype == kF32)
    linear_t<float>(L, x, stride);
  else if (x_dtype == kF16)
    linear_t<_Float16>(L, x, stride);
  else
    linear_t<__bf16>(L, x, stride);
  return hipGetLastError();
}

bool mx_matmul_fits(int rows, int cols, int batch) { return !mx_wants_gemm(rows, cols, batch) || mx_gemm_fits(rows, cols, batch); }

size_t mx_matmul_workspace(int rows, int cols, int batch) {
  return mx_wants_gemm(rows, cols, batch) ? mx_gemm_workspace(rows, cols, batch) : 0;
}

hipError_t launch_mx_matmul(const MxMatmul& L) {
  if (mx_wants_gemm(L.rows, L.cols, L.batch)) return launch_mx_gemm(L);
  const int tokens = (L.batch + 15) / 16, tiles = (L.rows + 15) / 16;
  if (tokens == 1)
    matvec_t<void>(L, 0, nullptr, 0, 0);
  else
    hipLaunchKernelGGL((mx_matvec_kernel<4, 2, 4, void>), dim3(mx_matvec_grid(tiles), (tokens + 3) / 4), dim3(256), 0,
                       L.stream, L, tiles, (const void*)nullptr, (int64_t)0, 0);
  return hipGetLastError();
}

}  // namespace nrq
