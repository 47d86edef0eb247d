// Rotary positions, and the same with the append of keys and values to a paged
// cache (include/nrq_serve.h, nrq_dev_rope and nrq_dev_rope_append).
//
// Pair i of every head of token t turns by a = pos[t] * freqs[i]. The product
// has up to 55 significant bits and a reaches 2^31 radians, so it is formed and
// reduced to a quarter turn in f64; sine and cosine of the rest, in [-pi/4,
// pi/4], are Taylor sums in f32 (the dropped terms are below 2^-29).
// The angles are shared by all heads: a workgroup takes a few tokens, forms
// their table once in LDS and then streams the heads through it, 16 bytes a lane.
#include "nrq_page.h"
#include "nrq_serve_launch.h"

namespace nrq {
namespace {

constexpr int kRopeNT = 256;
constexpr int kRopePairs = 512;  // pairs of the tokens of a workgroup: 4 KiB of LDS

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

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// One head of one token: where its row comes from and goes to. kind 0: q, 1: k, 2: v.
template <typename T>
struct RopeRow {
  const T* src;
  T* y;         // q
  uint16_t* c;  // k, v: the cache row, nullptr if there is none
};

template <typename T, typename C, int V>
__device__ __forceinline__ void rope_put(const RopeRow<T>& r, int d, const float* f) {
  if (r.y) {
    Vec<T, V> o;
#pragma unroll
    for (int i = 0; i < V; i++) o.v[i] = (T)f[i];
    *(Vec<T, V>*)(r.y + d) = o;
  } else if (r.c) {
    Vec<C, V> o;
#pragma unroll
    for (int i = 0; i < V; i++) o.v[i] = (C)f[i];
    *(Vec<C, V>*)((C*)r.c + d) = o;
  }
}

// T: the rows' type, C: the cache's, V: elements of one access (16 bytes of T
// where strides, addresses and the rotated part allow it, else 1 or, for
// adjacent pairs, 2 by scalar accesses).
template <typename T, typename C, int V, bool APPEND>
__global__ __launch_bounds__(kRopeNT) void rope_kernel(RopeLaunch L, int tpw) {
  __shared__ float2 cs[kRopePairs];
  const int t0 = blockIdx.x * tpw, nt = min(tpw, L.tokens - t0);
  for (int i = threadIdx.x; i < nt * L.nf; i += kRopeNT) {
    const float2 v = sincos_turn(L.pos[t0 + i / L.nf], L.freqs[i % L.nf]);
    cs[i] = make_float2(v.x * L.scale, v.y * L.scale);
  }
  __syncthreads();
  const int heads = APPEND ? L.heads + 2 * L.kv.n_kv : L.heads;
  const int half = L.nf, rot = 2 * half;
  // items of a head: with NEOX pairs an access of each half, else one access; then the rest of the head
  const int rest0 = rot / V, chunks = L.hd / V;
  const int pairs = L.neox ? half / V : (V == 1 ? half : rest0);  // items that rotate
  const int items = pairs + chunks - rest0;
  const int per_token = heads * items, total = nt * per_token;
  const int step = kRopeNT * gridDim.y;
  for (int it = blockIdx.y * kRopeNT + threadIdx.x; it < total; it += step) {
    const int tt = it / per_token, r = it - tt * per_token, h = r / items, c = r - h * items;
    const int t = t0 + tt;
    RopeRow<T> row;
    row.y = nullptr;
    row.c = nullptr;
    bool turn = true;
    if (!APPEND) {
      row.src = (const T*)L.x + t * L.xt + h * L.xh;
      row.y = (T*)L.y + t * L.yt + h * L.yh;
    } else {
      const int seq = L.seq[t], pos = L.pos[t];
      if (seq < 0 || seq >= L.table.seqs || pos < 0) continue;  // padding
      if (h < L.heads) {
        row.src = (const T*)L.x + t * L.xt + h * L.xh;
        row.y = (T*)L.y + t * L.yt + h * L.yh;
      } else {
        const bool isk = h < L.heads + L.kv.n_kv;
        const int hh = h - L.heads - (isk ? 0 : L.kv.n_kv);
        const uint32_t place = page_place(L.table.pages + seq * L.table.stride, L.table.width, L.kv.page_size,
                                          L.kv.n_pages, L.kv.page_stride8, L.kv.pos_stride8, pos);
        if (place == kNoPlace) continue;
        row.src = isk ? (const T*)L.k + t * L.kt + hh * L.kh : (const T*)L.v + t * L.vt + hh * L.vh;
        row.c = (isk ? L.kv.k : L.kv.v) + (uint64_t)place * 8 + hh * L.kv.head_stride;
        turn = isk;
      }
    }
    const float2* w = cs + tt * half;
    if (c >= pairs) {  // behind the rotated part
      const int d = (rest0 + c - pairs) * V;
      const Vec<T, V> a = *(const Vec<T, V>*)(row.src + d);
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i++) o[i] = (float)a.v[i];
      rope_put<T, C, V>(row, d, o);
    } else if (L.neox) {
      const int d = c * V;
      const Vec<T, V> a = *(const Vec<T, V>*)(row.src + d), b = *(const Vec<T, V>*)(row.src + d + half);
      float o0[V], o1[V];
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float x0 = (float)a.v[i], x1 = (float)b.v[i];
        const float2 k = turn ? w[d + i] : make_float2(1.0f, 0.0f);
        o0[i] = turn ? fmaf(x0, k.x, -(x1 * k.y)) : x0;
        o1[i] = turn ? fmaf(x0, k.y, x1 * k.x) : x1;
      }
      rope_put<T, C, V>(row, d, o0);
      rope_put<T, C, V>(row, d + half, o1);
    } else {
      constexpr int P = V == 1 ? 2 : V;  // scalar accesses: the item is one pair
      const int d = V == 1 ? 2 * c : c * V;
      T x[P];
      if constexpr (V == 1) {
        x[0] = row.src[d];
        x[1] = row.src[d + 1];
      } else {
        const Vec<T, V> a = *(const Vec<T, V>*)(row.src + d);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = a.v[i];
      }
      float o[P];
#pragma unroll
      for (int i = 0; i < P; i += 2) {
        const float x0 = (float)x[i], x1 = (float)x[i + 1];
        const float2 k = w[(d + i) >> 1];
        o[i] = turn ? fmaf(x0, k.x, -(x1 * k.y)) : x0;
        o[i + 1] = turn ? fmaf(x0, k.y, x1 * k.x) : x1;
      }
      if constexpr (V == 1) {
        rope_put<T, C, 1>(row, d, o);
        rope_put<T, C, 1>(row, d + 1, o + 1);
      } else {
        rope_put<T, C, V>(row, d, o);
      }
    }
  }
}

template <typename T, typename C, bool APPEND>
hipError_t launch_t(const RopeLaunch& L) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](const void* p, int64_t s0, int64_t s1) {
    return ((uintptr_t)p & 15) == 0 && s0 % V == 0 && s1 % V == 0;
  };
  bool wide = fits(L.x, L.xt, L.xh) && fits(L.y, L.yt, L.yh) && L.hd % V == 0 && (L.neox ? L.nf : 2 * L.nf) % V == 0;
  if (APPEND) wide = wide && fits(L.k, L.kt, L.kh) && fits(L.v, L.vt, L.vh);
  // tokens of a workgroup: as many as make one angle a thread
  const int tpw = L.nf > kRopeNT ? 1 : kRopeNT / L.nf;
  const int t = tpw < L.tokens ? tpw : L.tokens;
  const int64_t work = (int64_t)t * (L.heads + (APPEND ? 2 * L.kv.n_kv : 0)) * L.hd;
  const int tw = (L.tokens + t - 1) / t;
  // few tokens: their heads are spread over more workgroups, at least an access a thread in each
  int64_t gy = tw >= 512 ? 1 : (512 + tw - 1) / tw;
  if (gy * kRopeNT * V > work) gy = work < kRopeNT * V ? 1 : work / (kRopeNT * V);
  const dim3 grid(tw, (unsigned)gy);
  if (wide)
    hipLaunchKernelGGL((rope_kernel<T, C, V, APPEND>), grid, dim3(kRopeNT), 0, L.stream, L, t);
  else
    hipLaunchKernelGGL((rope_kernel<T, C, 1, APPEND>), grid, dim3(kRopeNT), 0, L.stream, L, t);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_c(const RopeLaunch& L) {
  if (!L.k) return launch_t<T, _Float16, false>(L);
  return L.kv.dtype == kF16 ? launch_t<T, _Float16, true>(L) : launch_t<T, __bf16, true>(L);
}

}  // namespace

hipError_t launch_rope(const RopeLaunch& L) {
  if (L.dtype == kF32) return launch_c<float>(L);
  if (L.dtype == kF16) return launch_c<_Float16>(L);
  return launch_c<__bf16>(L);
}

}  // namespace nrq
