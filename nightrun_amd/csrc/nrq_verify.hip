// Verification of drafted tokens (include/nrq_serve.h, nrq_dev_verify_drafts).
//
// Per sequence one row decides: the first refused draft's, or the one behind the
// last draft. The first launch finds it (a few gathers and a ballot, done again
// by every workgroup, which takes a run of spans so that this is not most of its time) and sums its
// weights over spans of 1024 tokens, the second adds the spans up, finds the one in which the drawn point lies and scans
// it. All sums are f64 in a fixed order: cumulative sums of 10^5 f32 weights in
// f32 would be off by more than the gap between neighbouring tokens. The deciding row is read once but for the span
// of the drawn point: 64 sequences over a vocabulary of 151,936 (78 MB of target's and draft's rows)
// take 21 us, 3.7 TB/s; one sequence 11 us, which is two launches and the gathers before them.
#include "nrq_serve_launch.h"

#include <climits>

namespace nrq {
namespace {

constexpr int kVerNT = 256;
constexpr int kVerPer = 4;                  // values of a thread: 16 bytes
constexpr int kVerSpan = kVerNT * kVerPer;  // values of a span
constexpr int kVerMost = 32;                // spans of a workgroup at most
constexpr int kVerFill = 2048;              // workgroups that the card holds

struct VerArgs {
  VerifyLaunch L;
  double* sums;  // [seqs][spans]
  int* counts;   // [seqs]: drafts accepted
  int spans, per;  // of a row, of a workgroup
};

struct VerRow {
  const float *p, *q;  // q: nullptr when the row is drawn from as it is
  int count;           // drafts accepted
  int n;               // drafts
  int without;         // certain drafts: the token left out, else -1
};

__device__ __forceinline__ VerRow verify_row(const VerifyLaunch& L, int b) {
  const int lane = threadIdx.x & 63;
  const int n = L.counts ? min(max(L.counts[b], 0), L.n_new) : L.n_new;
  bool ok = false;
  int d = -1;
  if (lane < n) {
    d = L.drafted[(int64_t)b * L.n_new + lane];
    if (d >= 0 && d < L.vocab) {
      const float p = L.target[b * L.tb + lane * L.tr + d];
      const float q = L.draft ? L.draft[b * L.db + lane * L.dr + d] : 1.0f;
      const float u = L.uniforms[(int64_t)b * (L.n_new + 1) + lane];
      ok = (double)u * (double)q < (double)p;  // exact: 48 bits
    }
  }
  const unsigned long long refused = ~__ballot(ok);
  VerRow r;
  r.n = n;
  r.count = refused ? min(n, __ffsll(refused) - 1) : n;
  r.p = L.target + b * L.tb + r.count * L.tr;
  r.q = r.count < n && L.draft ? L.draft + b * L.db + r.count * L.dr : nullptr;
  r.without = -1;
  if (r.count < n && !L.draft) {
    const int dd = __shfl(d, r.count);
    r.without = dd;
  }
  return r;
}

// weight of value v; NaN and negative ones are none
__device__ __forceinline__ double ver_weight(const VerRow& r, float p, float q, int v) {
  if (r.q) {
    const double diff = (double)p - (double)q;
    return diff > 0.0 ? diff : 0.0;
  }
  return p > 0.0f && v != r.without ? (double)p : 0.0;
}

__device__ __forceinline__ void ver_load(const VerRow& r, int v0, int vocab, float* p, float* q) {
  const bool wide = v0 + kVerPer <= vocab && (((uintptr_t)r.p | (uintptr_t)r.q) & 15) == 0;
  if (wide) {
    const float4 a = *(const float4*)(r.p + v0), c = r.q ? *(const float4*)(r.q + v0) : make_float4(0, 0, 0, 0);
    p[0] = a.x, p[1] = a.y, p[2] = a.z, p[3] = a.w;
    q[0] = c.x, q[1] = c.y, q[2] = c.z, q[3] = c.w;
  } else {
#pragma unroll
    for (int i = 0; i < kVerPer; i++) {
      p[i] = v0 + i < vocab ? r.p[v0 + i] : 0.0f;
      q[i] = r.q && v0 + i < vocab ? r.q[v0 + i] : 0.0f;
    }
  }
}

// Sum over the wave, in a fixed order.
__device__ __forceinline__ double ver_wave_sum(double s) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
  return s;
}

__global__ __launch_bounds__(kVerNT) void verify_sums_kernel(VerArgs A) {
  __shared__ double part[kVerMost][kVerNT / 64];
  const int b = blockIdx.y, s0 = blockIdx.x * A.per, s1 = min(s0 + A.per, A.spans), t = threadIdx.x;
  const VerRow r = verify_row(A.L, b);
  if (s0 == 0 && t == 0) A.counts[b] = r.count;
  float p[kVerPer], q[kVerPer], pn[kVerPer] = {0, 0, 0, 0}, qn[kVerPer] = {0, 0, 0, 0};
  ver_load(r, s0 * kVerSpan + t * kVerPer, A.L.vocab, p, q);
  for (int k = s0; k < s1; k++) {  // the next span is on its way while this one is added up
    const int v0 = k * kVerSpan + t * kVerPer;
    if (k + 1 < s1) ver_load(r, v0 + kVerSpan, A.L.vocab, pn, qn);
    double s = 0;
#pragma unroll
    for (int i = 0; i < kVerPer; i++)
      if (v0 + i < A.L.vocab) s += ver_weight(r, p[i], q[i], v0 + i);
    s = ver_wave_sum(s);
    if ((t & 63) == 0) part[k - s0][t >> 6] = s;
#pragma unroll
    for (int i = 0; i < kVerPer; i++) p[i] = pn[i], q[i] = qn[i];
  }
  __syncthreads();
  if (t < s1 - s0) {
    double s = 0;
    for (int w = 0; w < kVerNT / 64; w++) s += part[t][w];
    A.sums[(int64_t)b * A.spans + s0 + t] = s;
  }
}

// Sums over the workgroup's threads up to and before each. The lanes add in different orders, so that the sums need
// not grow with the thread to the last bit, not even behind the last weight: more than one thread may find a point
// between its two. Who draws is the first thread with weight whose `upto` is above the point, and that one alone.
struct VerSum {
  double before, upto, total;
};
__device__ __forceinline__ VerSum ver_scan(double own, double* lds) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double x = own;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  if (lane == 63) lds[w] = x;
  double y = __shfl_up(x, 1);
  if (lane == 0) y = 0;
  __syncthreads();
  double before = 0, all = 0;
  for (int i = 0; i < kVerNT / 64; i++) {
    if (i == w) before = all;
    all += lds[i];
  }
  return VerSum{before + y, before + x, all};
}

// The workgroup's first thread for which `on` holds, kVerNT if there is none.
__device__ __forceinline__ int ver_first(bool on, int* lds) {
  const int w = threadIdx.x >> 6;
  const unsigned long long m = __ballot(on);
  if ((threadIdx.x & 63) == 0) lds[w] = m ? 64 * w + __ffsll(m) - 1 : kVerNT;
  __syncthreads();
  int t = kVerNT;
#pragma unroll
  for (int i = 0; i < kVerNT / 64; i++) t = min(t, lds[i]);
  return t;
}

__global__ __launch_bounds__(kVerNT) void verify_draw_kernel(VerArgs A) {
  __shared__ double lds[3][kVerNT / 64], base;
  __shared__ int first[2][kVerNT / 64], found, last[2], drawn;
  const VerifyLaunch& L = A.L;
  const int b = blockIdx.x, t = threadIdx.x;
  double* sums = A.sums + (int64_t)b * A.spans;
  // each thread adds up a run of spans (one, up to 262144 tokens)
  const int per = (A.spans + kVerNT - 1) / kVerNT, s0 = min(t * per, A.spans), s1 = min(s0 + per, A.spans);
  double own = 0;
  for (int i = s0; i < s1; i++) own += sums[i];
  const int n = L.counts ? min(max(L.counts[b], 0), L.n_new) : L.n_new;
  VerRow r;
  r.count = A.counts[b];
  r.p = L.target + b * L.tb + r.count * L.tr;
  r.q = r.count < n && L.draft ? L.draft + b * L.db + r.count * L.dr : nullptr;
  r.without = r.count < n && !L.draft ? L.drafted[(int64_t)b * L.n_new + r.count] : -1;
  const double drawn_u = (double)L.uniforms[(int64_t)b * (L.n_new + 1) + L.n_new], u = drawn_u < 0.0 ? 0.0 : drawn_u;
  if (t == 0) found = drawn = -1;
  if (t < 2) last[t] = -1;
  VerSum c = ver_scan(own, lds[0]);
  if (!(c.total > 0.0) && (r.q || r.without >= 0)) {  // nothing left: the target itself (rare, by this workgroup alone)
    r.q = nullptr;
    r.without = -1;
    own = 0;
    for (int i = s0; i < s1; i++) {
      double s = 0;
      for (int v = i * kVerSpan; v < min((i + 1) * kVerSpan, L.vocab); v++) s += ver_weight(r, r.p[v], 0.0f, v);
      sums[i] = s;  // read again by this thread only
      own += s;
    }
    c = ver_scan(own, lds[1]);
  }
  // the first span with weight whose cumulative sum is above the point; a uniform of 1 has none (its product with
  // the sum may be an ulp below what another lane's order gives)
  const double point = u < 1.0 ? u * c.total : INFINITY;
  if (t == ver_first(own > 0.0 && c.upto > point, first[0])) {
    double before = c.before;
    int at = -1;
    for (int i = s0; i < s1; i++) {
      const double s = sums[i];
      if (!(s > 0.0)) continue;
      at = i;
      base = before;
      if (before + s > point) break;
      before += s;
    }
    found = at;  // where rounding leaves the point behind the run, its last span with weight
  }
  __syncthreads();
  int span = found;
  const bool past = span < 0;
  if (past) {  // no sum is above the point (a uniform of 1, or no weight): the last span with any
    for (int i = s0; i < s1; i++)
      if (sums[i] > 0.0) atomicMax(&last[0], i);
    __syncthreads();
    span = last[0];
  }
  int token = -1;
  if (span >= 0) {
    const int v0 = span * kVerSpan + t * kVerPer;
    double w[kVerPer], s = 0;
    float p[kVerPer], q[kVerPer];
    ver_load(r, v0, L.vocab, p, q);
#pragma unroll
    for (int i = 0; i < kVerPer; i++) {
      w[i] = v0 + i < L.vocab ? ver_weight(r, p[i], q[i], v0 + i) : 0.0;
      s += w[i];
    }
    const VerSum e = ver_scan(s, lds[2]);
    const double point1 = past ? INFINITY : point - base;
    int lastw = -1;
#pragma unroll
    for (int i = 0; i < kVerPer; i++)
      if (w[i] > 0.0) lastw = v0 + i;
    if (t == ver_first(s > 0.0 && e.upto > point1, first[1])) {
      double at = e.before;
      int v = -1;
#pragma unroll
      for (int i = 0; i < kVerPer; i++) {
        at += w[i];
        if (v < 0 && w[i] > 0.0 && at > point1) v = v0 + i;
      }
      drawn = v < 0 ? lastw : v;  // the scan's rounding and this sum's may differ
    }
    __syncthreads();
    token = drawn;
    if (token < 0) {  // past the last weight, or what the span's sums differ by
      if (lastw >= 0) atomicMax(&last[1], lastw);
      __syncthreads();
      token = last[1];
    }
  }
  if (t == 0) L.accepted[b] = r.count;
  for (int j = t; j <= L.n_new; j += kVerNT)
    L.tokens[(int64_t)b * (L.n_new + 1) + j] =
        j < r.count ? L.drafted[(int64_t)b * L.n_new + j] : (j == r.count ? token : -1);
}

}  // namespace

size_t verify_workspace(size_t seqs, size_t vocab) {
  return seqs * ((vocab + kVerSpan - 1) / kVerSpan * sizeof(double) + sizeof(int));
}

hipError_t launch_verify(const VerifyLaunch& L) {
  const int spans = (L.vocab + kVerSpan - 1) / kVerSpan;
  VerArgs A{L, (double*)L.workspace, (int*)((double*)L.workspace + (size_t)L.seqs * spans), spans, 1};
  // as many workgroups as the card holds, with equal runs of spans
  int groups = kVerFill / L.seqs;
  if (groups < (spans + kVerMost - 1) / kVerMost) groups = (spans + kVerMost - 1) / kVerMost;
  A.per = (spans + groups - 1) / groups;
  for (int b0 = 0; b0 < L.seqs; b0 += 65535) {  // gridDim.y
    VerArgs P = A;
    const int n = L.seqs - b0 < 65535 ? L.seqs - b0 : 65535;
    P.L.tokens += (int64_t)b0 * (L.n_new + 1);
    P.L.accepted += b0;
    P.L.target += b0 * L.tb;
    if (L.draft) P.L.draft += b0 * L.db;
    P.L.drafted += (int64_t)b0 * L.n_new;
    P.L.uniforms += (int64_t)b0 * (L.n_new + 1);
    if (L.counts) P.L.counts += b0;
    P.sums += (int64_t)b0 * A.spans;
    P.counts += b0;
    hipLaunchKernelGGL(verify_sums_kernel, dim3((A.spans + A.per - 1) / A.per, n), dim3(kVerNT), 0, L.stream, P);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(n), dim3(kVerNT), 0, L.stream, P);
  }
  return hipGetLastError();
}

}  // namespace nrq
