// MXFP4 (include/nrq_serve.h): quantization, its inverse, and the product of
// two quantized matrices on the scaled matrix instructions.
//
// v_mfma_scale_f32_16x16x128 takes from lane l the 32 values of one block: row
// l % 16 of its operand, columns 32 (l / 16) .. + 31 of the step's 128, 16
// consecutive bytes of the row, and the block's scale byte. The product of two
// values has at most 4 significant bits, so the sums within a block are exact.
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

// Eight values of a row: 16 bytes or, for unaligned rows, one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float* f) {
  constexpr int V = 16 / sizeof(T);
  if (wide) {
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

template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* src, int64_t stride, uint32_t cols8, int64_t items,
                                                          uint32_t* q, uint8_t* sc, int wide) {
  // grid-stride over groups of 8 values; four lanes a block, and the grid's size
  // is a multiple of four, so a block's lanes stay together
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / cols8;
    const int c = (int)(i - row * cols8) * 8;
    float f[8];
    load8(src + row * stride + c, wide, f);
    uint32_t s;
    q[i] = mx_quantize8(f, &s);
    if ((threadIdx.x & 3) == 0) sc[i >> 2] = (uint8_t)s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* q, const uint8_t* sc, int64_t stride,
                                                            uint32_t cols8, int64_t items, T* dst, int wide) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / cols8;
    const int c = (int)(i - row * cols8) * 8;
    const uint32_t w = q[i], s = sc[i >> 2];
    const float by = __uint_as_float(s == 255u ? 0x7fc00000u : (s ? s << 23 : 0x00400000u));
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      // code eem of 2^(ee - 1) (1 + m / 2), or m / 2: times 4 an integer
      const uint32_t n = (w >> (4 * k)) & 15u, ee = (n >> 1) & 3u, m = n & 1u;
      const float mag = ee ? __uint_as_float(((ee + 126u) << 23) | (m << 22)) : 0.5f * m;
      f[k] = (n & 8u ? -mag : mag) * by;
    }
    T* d = dst + row * stride + c;
    constexpr int V = 16 / sizeof(T);
    if (wide) {
#pragma unroll
      for (int k = 0; k < 8; k += V) {
        Half16<T> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.v[j] = (T)f[k + j];
        *(Half16<T>*)(d + k) = o;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) d[k] = (T)f[k];
    }
  }
}

// One lane's block: 16 bytes and its scale; zeros with scale 1 for none.
struct MxBlock {
  i32x4 q;
  int s;
};
__device__ __forceinline__ MxBlock mx_block(const uint8_t* q, const uint8_t* s, bool live) {
  MxBlock b;
  b.q = live ? *(const i32x4*)q : i32x4{0, 0, 0, 0};
  b.s = live ? (int)*s : 127;
  return b;
}

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

// 16 rows of w times 16 NT tokens per workgroup; its four waves take every
// fourth step of 128 columns, then add up in LDS.
template <int NT>
__global__ __launch_bounds__(256) void mx_matvec_kernel(MxMatmul L) {
  __shared__ f32x4 part[3][NT][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, steps = (blocks + 3) / 4;
  const int row = blockIdx.x * 16 + i;
  const uint8_t* wq = L.w + (int64_t)min(row, L.rows - 1) * blocks * 16;
  const uint8_t* wsc = L.ws + (int64_t)min(row, L.rows - 1) * blocks;
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) acc[t] = f32x4{0, 0, 0, 0};
  for (int s = w; s < steps; s += 4) {
    const int b = 4 * s + g;
    const MxBlock a = mx_block(wq + (int64_t)b * 16, wsc + b, b < blocks && row < L.rows);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int tok = (blockIdx.y * NT + t) * 16 + i;
      const int64_t at = (int64_t)tok * blocks + b;
      acc[t] = mx_mfma(a, mx_block(L.x + at * 16, L.xs + at, b < blocks && tok < L.batch), acc[t]);
    }
  }
  if (w)
#pragma unroll
    for (int t = 0; t < NT; t++) part[w - 1][t][lane] = acc[t];
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    acc[t] += part[0][t][lane];
    acc[t] += part[1][t][lane];
    acc[t] += part[2][t][lane];
    const int tok = (blockIdx.y * NT + t) * 16 + i, r = blockIdx.x * 16 + 4 * g;
    if (tok < L.batch && r < L.rows) mx_store(L.y, L.dtype, tok * L.ldy + r, L.rows - r, acc[t]);
  }
}

template <typename T>
bool wide_rows(const void* p, int64_t stride) {
  return ((uintptr_t)p & 15) == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
}

template <typename T>
void quantize_t(const void* src, size_t rows, size_t cols, int64_t stride, void* q, void* s, hipStream_t st) {
  const int64_t items = (int64_t)rows * (cols / 8);
  const unsigned grid = (unsigned)(items + 255 < 256 * (int64_t)8192 ? (items + 255) / 256 : 8192);
  hipLaunchKernelGGL((mx_quantize_kernel<T>), dim3(grid), dim3(256), 0, st, (const T*)src, stride, (uint32_t)(cols / 8),
                     items, (uint32_t*)q, (uint8_t*)s, wide_rows<T>(src, stride) ? 1 : 0);
}

template <typename T>
void dequantize_t(const void* q, const void* s, size_t rows, size_t cols, void* dst, int64_t stride, hipStream_t st) {
  const int64_t items = (int64_t)rows * (cols / 8);
  const unsigned grid = (unsigned)(items + 255 < 256 * (int64_t)8192 ? (items + 255) / 256 : 8192);
  hipLaunchKernelGGL((mx_dequantize_kernel<T>), dim3(grid), dim3(256), 0, st, (const uint32_t*)q, (const uint8_t*)s,
                     stride, (uint32_t)(cols / 8), items, (T*)dst, wide_rows<T>(dst, stride) ? 1 : 0);
}

}  // namespace

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

hipError_t launch_mx_matmul(const MxMatmul& L) {
  if (L.batch > 64 && L.cols >= 64) return launch_mx_gemm(L);
  const int tiles = (L.batch + 15) / 16;
  const unsigned gx = (unsigned)((L.rows + 15) / 16);
  if (tiles == 1)
    hipLaunchKernelGGL((mx_matvec_kernel<1>), dim3(gx), dim3(256), 0, L.stream, L);
  else
    hipLaunchKernelGGL((mx_matvec_kernel<4>), dim3(gx, (tiles + 3) / 4), dim3(256), 0, L.stream, L);
  return hipGetLastError();
}

}  // namespace nrq
