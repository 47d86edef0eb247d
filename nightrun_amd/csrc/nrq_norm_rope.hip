// Norms of queries and keys for each head with the rotary positions in the same pass, and the same with the
// append of keys and values to a paged cache (include/nrq_tree.h, nrq_dev_norm_rope and nrq_dev_norm_rope_append).
//
// A row (one head of one token) is held by a group of lanes, a power of two of them, from its load over the sum of its
// squares and the rotation to its store, so that memory sees each value once each way. As without the norm
// (nrq_rope.hip) a workgroup takes a few tokens, forms their angles once in LDS and goes through their rows; an item is an access
// of the row, with NEOX pairs one of each half, so that a pair is always in one lane. The first rows are asked for
// before the angles are formed, and each turn's while the turn before it is finished.
//
// Memory bounds it: 16,381 tokens of 33 heads of 128 in f16 (277 MB both ways, read and written once as the counters show)
// take 60 to 64 us, 4.5 TB/s (93 without the rows of the next turn on their way and with the sums through LDS). 1536 nodes of 32 + 8 + 8
// heads into a bf16 cache (38 MB) take 14.3 us, twice what their bytes do: a workgroup has two turns, the second of them half empty, and before
// them positions, pages and angles. The append of a prompt of 4096 (101 MB) takes 23.1, 4.4 TB/s; two of its registers spill under the bound of
// four waves a SIMD (bf16 and f16 rows). One token takes as long as a launch does.
//
// Rows that do not go in accesses of 16 bytes (pointers, strides, or a rotated part that ends inside one: with f16 rows and NEOX pairs one
// of 40 dimensions, say) take several times as long: one value an access, one row of a lane in flight, and sixteen places for items, as
// rows of 1024 need, of which a head of 128 fills two. 16,381 tokens of 32 heads of 128, f16, 40 dimensions rotated: 515 us, where
// all 128 take 48; heads of 96 with 24 of them 461; the append of 4096 tokens 225. Without norms (a place of its own for each token)
// that append takes 128, and 70 in nrq_rope.hip, which takes no such places and keeps four rows in flight.
#include "nrq_page.h"
#include "nrq_tree_launch.h"
#include "nrq_turn.h"

namespace nrq {
namespace {

constexpr int kNrNT = 256;
constexpr int kNrPairs = 512;  // pairs of the tokens of a workgroup: 4 KiB of LDS
constexpr int kNrTokens = 64;  // tokens of a workgroup at most

struct NrArgs {
  NormRopeLaunch L;
  int tpw;     // tokens of a workgroup
  int lanes;   // of a row: a power of two, at most 64
  int pairs;   // items that rotate
  int items;   // of a row
  float inv;   // 1 / head_dim
};

// Where a row comes from and goes to, and its values: d and d1 of the lane's items.
template <typename T, int V, int K>
struct NrRow {
  Vec<T, V> a[K], b[K];
  void* to;  // nullptr: nowhere
  int kind;  // 0: q, 1: k, 2: v
  int tok;
};

// The sum over a group of lanes, a power of two of them, the same in each. A lane whose quad has one sum finds the
// other quad's mirrored in the eight lanes, and so on.
template <int CTRL>
__device__ __forceinline__ float nr_dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 15, 15, true));
}
__device__ __forceinline__ float nr_sum(float s, int lanes) {
  if (lanes > 1) s += nr_dpp<0xb1>(s);   // the neighbour in a pair
  if (lanes > 2) s += nr_dpp<0x4e>(s);   // the other pair of a quad
  if (lanes > 4) s += nr_dpp<0x141>(s);  // mirrored in eight lanes
  if (lanes > 8) s += nr_dpp<0x140>(s);  // mirrored in sixteen
  if (lanes > 16) s += __shfl_xor(s, 16);
  if (lanes > 32) s += __shfl_xor(s, 32);
  return s;
}

// T: the rows' type, C: the cache's, V: elements of an access (16 bytes of T, or 1 where strides, addresses
// or the rotated part do not allow it), K: items of a lane at most, A: rows of a lane in a turn, the next turn's on their way.
template <typename T, typename C, int V, int K, int A, bool APPEND, bool NORM>
__global__ __launch_bounds__(kNrNT, K == 1 && V > 1 ? 4 : 1) void norm_rope_kernel(NrArgs P) {
  __shared__ float2 cs[kNrPairs];
  __shared__ uint32_t place[kNrTokens];
  __shared__ bool pad[kNrTokens];
  const RopeLaunch& L = P.L.r;
  const int t0 = blockIdx.x * P.tpw, nt = min(P.tpw, L.tokens - t0), half = L.nf;
  const int heads = APPEND ? L.heads + 2 * L.kv.n_kv : L.heads;
  const int across = kNrNT / P.lanes, lane = threadIdx.x & (P.lanes - 1);
  const int step = across * gridDim.y, dt = step / heads, dh = step - dt * heads;
  // a lane's places in the row: the first access, and with pairs that lie apart the second
  const int rest0 = 2 * half;
  int d[K], d1[K];
  bool turning[K], two[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int c = lane + P.lanes * k;
    turning[k] = c < P.pairs;
    d[k] = !turning[k] ? rest0 + (c - P.pairs) * V : (L.neox ? c * V : (V == 1 ? 2 * c : c * V));
    two[k] = turning[k] && (L.neox || V == 1);
    d1[k] = two[k] ? (L.neox ? d[k] + half : d[k] + 1) : d[k];
  }
  int r = (int)threadIdx.x / P.lanes + across * blockIdx.y, tt = r / heads, h = r - tt * heads;
  // a turn's rows; also padding's, which are not stored
  auto fetch = [&](NrRow<T, V, K>* row) {
#pragma unroll
    for (int j = 0; j < A; j++) {
      NrRow<T, V, K>& w = row[j];
      const T* from = nullptr;
      w.kind = -1, w.tok = min(tt, nt - 1);
      const int t = t0 + tt;
      if (tt < nt) {
        if (!APPEND || h < L.heads) {
          w.kind = 0;
          from = (const T*)L.x + t * L.xt + h * L.xh;
          w.to = (T*)L.y + t * L.yt + h * L.yh;
        } else {
          const bool isk = h < L.heads + L.kv.n_kv;
          const int hh = h - L.heads - (isk ? 0 : L.kv.n_kv);
          w.kind = isk ? 1 : 2;
          from = isk ? (const T*)L.k + t * L.kt + hh * L.kh : (const T*)L.v + t * L.vt + hh * L.vh;
          w.to = (C*)(isk ? L.kv.k : L.kv.v) + hh * L.kv.head_stride;
        }
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        w.a[k] = w.b[k] = Vec<T, V>{};
        if (from && lane + P.lanes * k < P.items) {
          w.a[k] = *(const Vec<T, V>*)(from + d[k]);
          if (two[k]) w.b[k] = *(const Vec<T, V>*)(from + d1[k]);
        }
      }
      h += dh;
      tt += dt;
      if (h >= heads) h -= heads, tt++;
    }
  };
  NrRow<T, V, K> first[A], second[A];
  fetch(first);  // on their way while the angles are formed
  for (int i = threadIdx.x; i < nt * half; i += kNrNT) {
    const float2 v = sincos_turn(L.pos[t0 + i / half], L.freqs[i % half]);
    cs[i] = make_float2(v.x * L.scale, v.y * L.scale);
  }
  if (APPEND)
    for (int i = threadIdx.x; i < nt; i += kNrNT) {
      const int seq = L.seq[t0 + i], at = P.L.at ? P.L.at[t0 + i] : L.pos[t0 + i];
      const bool p = seq < 0 || seq >= L.table.seqs || at < 0;
      pad[i] = p;
      place[i] = p ? kNoPlace
                   : page_place(L.table.pages + seq * L.table.stride, L.table.width, L.kv.page_size, L.kv.n_pages,
                                L.kv.page_stride8, L.kv.pos_stride8, at);
    }
  // one item a lane: its weights stay in registers
  float wq[2][V], wk[2][V];
  if (NORM && K == 1 && lane < P.items) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      wq[0][i] = P.L.wq ? P.L.wq[d[0] + i] : 1.0f;
      wq[1][i] = P.L.wq ? P.L.wq[d1[0] + i] : 1.0f;
      if (APPEND) {
        wk[0][i] = P.L.wk ? P.L.wk[d[0] + i] : 1.0f;
        wk[1][i] = P.L.wk ? P.L.wk[d1[0] + i] : 1.0f;
      }
    }
  }
  __syncthreads();
  auto finish = [&](const NrRow<T, V, K>* row) {
#pragma unroll
    for (int j = 0; j < A; j++) {
      const NrRow<T, V, K>& w = row[j];
      float by = 1.0f;
      if (NORM) {  // all lanes of the wave
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
          for (int i = 0; i < V; i++) {
            const float x0 = (float)w.a[k].v[i], x1 = (float)w.b[k].v[i];  // zero without a second access
            s = fmaf(x0, x0, s);
            s = fmaf(x1, x1, s);
          }
        const float mean = nr_sum(s, P.lanes) * P.inv + P.L.eps;
        // the instruction is within a step of the value, but takes a subnormal mean for zero
        by = mean >= 0x1p-126f ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);
      }
      void* to = w.to;
      if (w.kind < 0) continue;
      if (APPEND) {
        if (w.kind == 0 ? pad[w.tok] : place[w.tok] == kNoPlace) continue;
        if (w.kind > 0) to = (C*)to + (uint64_t)place[w.tok] * 8;
      }
      const float2* cw = cs + w.tok * half;
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (lane + P.lanes * k >= P.items) continue;
        float o0[V], o1[V];
#pragma unroll
        for (int i = 0; i < V; i++) o0[i] = (float)w.a[k].v[i], o1[i] = (float)w.b[k].v[i];
        if (!APPEND || w.kind != 2) {
          if (NORM) {
            const bool isk = APPEND && w.kind == 1;
            const float* wt = isk ? P.L.wk : P.L.wq;
#pragma unroll
            for (int i = 0; i < V; i++) {
              float w0, w1;
              if (K == 1) {
                w0 = isk ? wk[0][i] : wq[0][i], w1 = isk ? wk[1][i] : wq[1][i];
              } else {
                w0 = wt ? wt[d[k] + i] : 1.0f, w1 = wt ? wt[d1[k] + i] : 1.0f;
              }
              o0[i] = o0[i] * by * w0, o1[i] = o1[i] * by * w1;
            }
          }
          if (two[k]) {
#pragma unroll
            for (int i = 0; i < V; i++) {
              const float2 q = cw[L.neox ? d[k] + i : d[k] / 2];
              const float x0 = o0[i], x1 = o1[i];
              o0[i] = fmaf(x0, q.x, -(x1 * q.y));
              o1[i] = fmaf(x0, q.y, x1 * q.x);
            }
          } else if (V > 1 && turning[k]) {
#pragma unroll
            for (int i = 0; i + 1 < V; i += 2) {
              const float2 q = cw[(d[k] + i) >> 1];
              const float x0 = o0[i], x1 = o0[i + 1];
              o0[i] = fmaf(x0, q.x, -(x1 * q.y));
              o0[i + 1] = fmaf(x0, q.y, x1 * q.x);
            }
          }
        }
        if (!APPEND || w.kind == 0) {
          Vec<T, V> v;
#pragma unroll
          for (int i = 0; i < V; i++) v.v[i] = (T)o0[i];
          *(Vec<T, V>*)((T*)to + d[k]) = v;
          if (two[k]) {
#pragma unroll
            for (int i = 0; i < V; i++) v.v[i] = (T)o1[i];
            *(Vec<T, V>*)((T*)to + d1[k]) = v;
          }
        } else {
          Vec<C, V> v;
#pragma unroll
          for (int i = 0; i < V; i++) v.v[i] = (C)o0[i];
          *(Vec<C, V>*)((C*)to + d[k]) = v;
          if (two[k]) {
#pragma unroll
            for (int i = 0; i < V; i++) v.v[i] = (C)o1[i];
            *(Vec<C, V>*)((C*)to + d1[k]) = v;
          }
        }
      }
    }
  };
  // every lane of a wave takes the same number of turns: the sums want all of them
  const int turns = (nt * heads + step * A - 1) / (step * A);
  for (int n = 0; n < turns; n += 2) {
    if (n + 1 < turns) fetch(second);
    finish(first);
    if (n + 1 >= turns) break;
    if (n + 2 < turns) fetch(first);
    finish(second);
  }
}

template <typename T, typename C, int V, int K, int A, bool APPEND, bool NORM>
hipError_t nr_launch(NrArgs& P) {
  const RopeLaunch& L = P.L.r;
  // Tokens of a workgroup: as many as make one angle a thread, fewer where fewer than 512 to 1024 workgroups would be
  // left (1536 nodes: 768 of them, 14.3 us; 18.4 with one token a workgroup); with few tokens their rows are spread over more workgroups, a row a group of lanes in each.
  int t = kNrNT / L.nf;
  t = t < 1 ? 1 : (t > kNrTokens ? kNrTokens : t);
  if (t > (L.tokens - 1) / 1024 + 1) t = (L.tokens - 1) / 1024 + 1;
  P.tpw = t;
  const int64_t rows = (int64_t)t * (L.heads + (APPEND ? 2 * L.kv.n_kv : 0)), across = kNrNT / P.lanes;
  const int tw = (L.tokens - 1) / t + 1;
  int64_t gy = tw >= 512 ? 1 : (512 + tw - 1) / tw;
  if (gy * across > rows) gy = rows < across ? 1 : rows / across;
  const int64_t most = (int64_t)t << 23;  // tokens of a launch: a grid has fewer than 2^32 threads
  for (int64_t t0 = 0; t0 < L.tokens; t0 += most) {
    NrArgs Q = P;
    RopeLaunch& R = Q.L.r;
    R.tokens = (int)(L.tokens - t0 < most ? L.tokens - t0 : most);
    R.x = (const T*)L.x + t0 * L.xt, R.y = (T*)L.y + t0 * L.yt, R.pos = L.pos + t0;
    if (APPEND) {
      R.k = (const T*)L.k + t0 * L.kt, R.v = (const T*)L.v + t0 * L.vt, R.seq = L.seq + t0;
      if (P.L.at) Q.L.at = P.L.at + t0;
    }
    const dim3 grid((R.tokens - 1) / t + 1, (unsigned)gy);
    hipLaunchKernelGGL((norm_rope_kernel<T, C, V, K, A, APPEND, NORM>), grid, dim3(kNrNT), 0, L.stream, Q);
  }
  return hipGetLastError();
}

template <typename T, typename C, bool APPEND, bool NORM>
hipError_t nr_launch_t(const NormRopeLaunch& N) {
  const RopeLaunch& L = N.r;
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](const void* p, int64_t s0, int64_t s1) {
    return ((uintptr_t)p & 15) == 0 && s0 % V == 0 && s1 % V == 0;
  };
  bool wide = fits(L.x, L.xt, L.xh) && fits(L.y, L.yt, L.yh) && L.hd % V == 0 && (L.neox ? L.nf : 2 * L.nf) % V == 0;
  if (APPEND) wide = wide && fits(L.k, L.kt, L.kh) && fits(L.v, L.vt, L.vh);
  NrArgs P;
  P.L = N;
  const int v = wide ? V : 1, rest0 = 2 * L.nf / v;
  P.pairs = L.neox ? L.nf / v : (v == 1 ? L.nf : rest0);
  P.items = P.pairs + L.hd / v - rest0;
  P.inv = 1.0f / (float)L.hd;
  P.lanes = 1;
  while (P.lanes < P.items && P.lanes < 64) P.lanes *= 2;
  // heads of 1024: 256 accesses of 4, or 1023 of 1 (where all but two dimensions are copied); the latter's kernel is
  // every row's that is not wide (at the file's head: what that costs)
  if (!wide) return nr_launch<T, C, 1, 16, 1, APPEND, NORM>(P);
  if (P.items <= 64) return nr_launch<T, C, V, 1, 2, APPEND, NORM>(P);
  return nr_launch<T, C, V, 4, 1, APPEND, NORM>(P);
}

template <typename T>
hipError_t nr_launch_c(const NormRopeLaunch& N) {
  if (!N.r.k) return nr_launch_t<T, _Float16, false, true>(N);
  if (N.r.kv.dtype == kF16) return N.norm ? nr_launch_t<T, _Float16, true, true>(N) : nr_launch_t<T, _Float16, true, false>(N);
  return N.norm ? nr_launch_t<T, __bf16, true, true>(N) : nr_launch_t<T, __bf16, true, false>(N);
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeLaunch& N) {
  if (N.r.dtype == kF32) return nr_launch_c<float>(N);
  if (N.r.dtype == kF16) return nr_launch_c<_Float16>(N);
  return nr_launch_c<__bf16>(N);
}

}  // namespace nrq
