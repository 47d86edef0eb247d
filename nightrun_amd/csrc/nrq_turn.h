// Sine and cosine of a rotary position's angle, for the kernels that rotate.
#pragma once

#include <hip/hip_runtime.h>

namespace nrq {
namespace {

// (cosine, sine) of pos * freq: the product and its reduction to a quarter turn in f64, the rest, in [-pi/4, pi/4],
// in Taylor sums in f32.
__device__ __forceinline__ float2 sincos_turn(int pos, float freq) {
  const double quarter = (double)pos * (double)freq * 0.63661977236758134308;  // 2 / pi
  const double n = rint(quarter);
  const float x = (float)(quarter - n) * 1.57079632679489662f;
  const int q = (int)(long long)n & 3;
  const float z = x * x;
  float s = fmaf(z, 1.0f / 362880, -1.0f / 5040);
  s = fmaf(z, s, 1.0f / 120);
  s = fmaf(z, s, -1.0f / 6);
  s = fmaf(x * z, s, x);
  float c = fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  c = fmaf(z, c, -1.0f / 720);
  c = fmaf(z, c, 1.0f / 24);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const float a = q & 1 ? s : c, b = q & 1 ? c : s;  // magnitudes of cosine and sine
  return make_float2(q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b);
}

// V values, one access
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

}  // namespace
}  // namespace nrq
