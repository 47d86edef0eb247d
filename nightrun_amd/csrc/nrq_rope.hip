// Rotary positions, and the same with the append of keys and values to a paged
// cache (include/nrq_serve.h, nrq_dev_rope and nrq_dev_rope_append).
//
// Pair i of every head of token t turns by a = pos[t] * freqs[i]. The product
// has up to 55 significant bits and a reaches 2^31 radians, so it is formed and
// reduced to a quarter turn in f64; sine and cosine of the rest, in [-pi/4,
// pi/4], are Taylor sums in f32 (the dropped terms are below 2^-29).
// The angles are shared by all heads: a workgroup takes a few tokens, forms
// their table once in LDS and then streams the heads through it, 16 bytes a lane.
// Memory bounds it: 4111 tokens of 40 heads of 128 in bf16 (84 MB both ways) take 17.8 us, 4.7 TB/s;
// 4096 new tokens of 32 + 8 + 8 heads of 64, f32 into an f16 cache (92 MB), 18.1 us, 5.1 TB/s. One
// token takes as long as a launch does.
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

constexpr int kRopeTokens = 64;  // tokens of a workgroup at most
constexpr int kRopeAhead = 4;    // rows of a thread whose loads are on their way together

// T: the rows' type, C: the cache's, V: elements of one access (16 bytes of T
// where strides, addresses and the rotated part allow it, else 1).
//
// An item is an access of one head's row (with NEOX pairs an access of each half), 256 / items
// rows at a time: a thread keeps its place in the row and goes from row to row.
template <typename T, typename C, int V, bool APPEND>
__global__ __launch_bounds__(kRopeNT) void rope_kernel(RopeLaunch L, int tpw) {
  __shared__ float2 cs[kRopePairs];
  __shared__ uint32_t place[kRopeTokens];
  __shared__ bool pad[kRopeTokens];
  const int t0 = blockIdx.x * tpw, nt = min(tpw, L.tokens - t0), half = L.nf;
  for (int i = threadIdx.x; i < nt * half; i += kRopeNT) {
    const float2 v = sincos_turn(L.pos[t0 + i / half], L.freqs[i % half]);
    cs[i] = make_float2(v.x * L.scale, v.y * L.scale);
  }
  if (APPEND)
    for (int i = threadIdx.x; i < nt; i += kRopeNT) {
      const int seq = L.seq[t0 + i], pos = L.pos[t0 + i];
      const bool p = seq < 0 || seq >= L.table.seqs || pos < 0;
      pad[i] = p;
      place[i] = p ? kNoPlace
                   : page_place(L.table.pages + seq * L.table.stride, L.table.width, L.kv.page_size, L.kv.n_pages,
                                L.kv.page_stride8, L.kv.pos_stride8, pos);
    }
  __syncthreads();
  const int heads = APPEND ? L.heads + 2 * L.kv.n_kv : L.heads;
  const int rest0 = 2 * half / V, chunks = L.hd / V;  // accesses of the rotated part, of a row
  const int pairs = L.neox ? half / V : (V == 1 ? half : rest0);  // items that rotate
  const int items = pairs + chunks - rest0;
  const int across = max(1, kRopeNT / items), lanes = min(items, kRopeNT);  // rows at a time; items over 256: one, in turns
  const int row0 = (int)threadIdx.x / lanes;
  if (row0 >= across) return;
  const int step = across * gridDim.y, dt = step / heads, dh = step - dt * heads;
  for (int c = (int)threadIdx.x - row0 * lanes; c < items; c += kRopeNT) {
    const bool turning = c < pairs;
    const int d = !turning ? (rest0 + c - pairs) * V : (L.neox ? c * V : (V == 1 ? 2 * c : c * V));
    const int d1 = !turning ? d : (L.neox ? d + half : d + 1);  // the second access, if any
    const bool two = turning && (L.neox || V == 1);
    int r = row0 + across * blockIdx.y, tt = r / heads, h = r - tt * heads;
    while (tt < nt) {
      Vec<T, V> a[kRopeAhead], b[kRopeAhead];
      const T* from[kRopeAhead];
      T* y[kRopeAhead];
      C* cache[kRopeAhead];
      int tok[kRopeAhead];
      bool turn[kRopeAhead];
#pragma unroll
      for (int k = 0; k < kRopeAhead; k++) {
        const int t = t0 + tt;
        bool on = tt < nt;
        tok[k] = tt;
        from[k] = nullptr;
        y[k] = nullptr;
        cache[k] = nullptr;
        turn[k] = turning;
        if (on) {
          if (!APPEND || h < L.heads) {
            on = !APPEND || !pad[tt];
            from[k] = (const T*)L.x + t * L.xt + h * L.xh;
            y[k] = (T*)L.y + t * L.yt + h * L.yh;
          } else {
            const bool isk = h < L.heads + L.kv.n_kv;
            const int hh = h - L.heads - (isk ? 0 : L.kv.n_kv);
            on = place[tt] != kNoPlace;
            from[k] = isk ? (const T*)L.k + t * L.kt + hh * L.kh : (const T*)L.v + t * L.vt + hh * L.vh;
            cache[k] = (C*)(isk ? L.kv.k : L.kv.v) + (uint64_t)place[tt] * 8 + hh * L.kv.head_stride;
            turn[k] = turning && isk;
          }
        }
        if (on) {
          a[k] = *(const Vec<T, V>*)(from[k] + d);
          if (two) b[k] = *(const Vec<T, V>*)(from[k] + d1);
        } else {
          from[k] = nullptr;
        }
        h += dh;
        tt += dt;
        if (h >= heads) h -= heads, tt++;
      }
#pragma unroll
      for (int k = 0; k < kRopeAhead; k++) {
        if (!from[k]) continue;
        const float2* w = cs + tok[k] * half;
        float o0[V], o1[V];
#pragma unroll
        for (int i = 0; i < V; i++) o0[i] = (float)a[k].v[i], o1[i] = two ? (float)b[k].v[i] : 0.0f;
        if (turn[k]) {
          if (two) {
#pragma unroll
            for (int i = 0; i < V; i++) {
              const float2 q = w[L.neox ? d + i : c];
              const float x0 = o0[i], x1 = o1[i];
              o0[i] = fmaf(x0, q.x, -(x1 * q.y));
              o1[i] = fmaf(x0, q.y, x1 * q.x);
            }
          } else if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
              const float2 q = w[(d + i) >> 1];
              const float x0 = o0[i], x1 = o0[i + 1];
              o0[i] = fmaf(x0, q.x, -(x1 * q.y));
              o0[i + 1] = fmaf(x0, q.y, x1 * q.x);
            }
          }
        }
        if (y[k]) {
          Vec<T, V> v;
#pragma unroll
          for (int i = 0; i < V; i++) v.v[i] = (T)o0[i];
          *(Vec<T, V>*)(y[k] + d) = v;
          if (two) {
#pragma unroll
            for (int i = 0; i < V; i++) v.v[i] = (T)o1[i];
            *(Vec<T, V>*)(y[k] + d1) = v;
          }
        } else {
          Vec<C, V> v;
#pragma unroll
          for (int i = 0; i < V; i++) v.v[i] = (C)o0[i];
          *(Vec<C, V>*)(cache[k] + d) = v;
          if (two) {
#pragma unroll
            for (int i = 0; i < V; i++) v.v[i] = (C)o1[i];
            *(Vec<C, V>*)(cache[k] + d1) = v;
          }
        }
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
  // Tokens of a workgroup: as many as make one angle a thread, fewer where the card (2048 workgroups) would not
  // be full; with few tokens their rows are spread over more workgroups, an access a thread in each.
  int t = kRopeNT / L.nf;
  t = t < 1 ? 1 : (t > kRopeTokens ? kRopeTokens : t);
  if (t > (L.tokens - 1) / 2048 + 1) t = (L.tokens - 1) / 2048 + 1;
  const int64_t work = (int64_t)t * (L.heads + (APPEND ? 2 * L.kv.n_kv : 0)) * L.hd;
  const int tw = (L.tokens - 1) / t + 1;
  int64_t gy = tw >= 512 ? 1 : (512 + tw - 1) / tw;
  if (gy * kRopeNT * V > work) gy = work < kRopeNT * V ? 1 : work / (kRopeNT * V);
  const int64_t most = (int64_t)t << 23;  // tokens of a launch: a grid has fewer than 2^32 threads
  for (int64_t t0 = 0; t0 < L.tokens; t0 += most) {
    RopeLaunch P = L;
    P.tokens = (int)(L.tokens - t0 < most ? L.tokens - t0 : most);
    P.x = (const T*)L.x + t0 * L.xt, P.y = (T*)L.y + t0 * L.yt, P.pos = L.pos + t0;
    if (APPEND) P.k = (const T*)L.k + t0 * L.kt, P.v = (const T*)L.v + t0 * L.vt, P.seq = L.seq + t0;
    const dim3 grid((P.tokens - 1) / t + 1, (unsigned)gy);
    if (wide)
      hipLaunchKernelGGL((rope_kernel<T, C, V, APPEND>), grid, dim3(kRopeNT), 0, L.stream, P, t);
    else
      hipLaunchKernelGGL((rope_kernel<T, C, 1, APPEND>), grid, dim3(kRopeNT), 0, L.stream, P, t);
  }
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
