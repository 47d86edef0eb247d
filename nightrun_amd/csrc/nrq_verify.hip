// Verification of drafted tokens (include/nrq_serve.h, nrq_dev_verify_drafts).
//
// Per sequence one row decides: the first refused draft's, or the one behind the
// last draft. The first launch finds it (a few gathers and a ballot, done again
// by every workgroup) and sums its weights over spans of the vocabulary, the
// second adds the spans up, finds the one in which the drawn point lies and scans
// it. All sums are f64 in a fixed order: cumulative sums of 10^5 f32 weights in
// f32 would be off by more than the gap between neighbouring tokens.
#include "nrq_serve_launch.h"

namespace nrq {
namespace {

constexpr int kVerNT = 256;
constexpr int kVerPer = 8;                     // values of a thread
constexpr int kVerSpan = kVerNT * kVerPer;     // values of a workgroup

struct VerArgs {
  VerifyLaunch L;
  double* sums;  // [seqs][spans][2]: of the residual, of the target
  int spans;
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

// weights of value v: of the residual and of the target; NaN and negative ones are none
__device__ __forceinline__ double2 ver_weight(const VerRow& r, float p, float q, int v) {
  const double tp = p > 0.0f ? (double)p : 0.0;
  double res = tp;
  if (r.q) {
    const double diff = (double)p - (double)q;
    res = diff > 0.0 ? diff : 0.0;
  } else if (v == r.without) {
    res = 0.0;
  }
  return make_double2(res, tp);
}

__device__ __forceinline__ void ver_load(const VerRow& r, int v0, int vocab, float* p, float* q) {
  const bool wide = v0 + kVerPer <= vocab && (((uintptr_t)r.p | (uintptr_t)r.q) & 15) == 0;
  if (wide) {
#pragma unroll
    for (int i = 0; i < kVerPer; i += 4) {
      const float4 a = *(const float4*)(r.p + v0 + i);
      const float4 c = r.q ? *(const float4*)(r.q + v0 + i) : make_float4(0, 0, 0, 0);
      p[i] = a.x, p[i + 1] = a.y, p[i + 2] = a.z, p[i + 3] = a.w;
      q[i] = c.x, q[i + 1] = c.y, q[i + 2] = c.z, q[i + 3] = c.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVerPer; i++) {
      p[i] = v0 + i < vocab ? r.p[v0 + i] : 0.0f;
      q[i] = r.q && v0 + i < vocab ? r.q[v0 + i] : 0.0f;
    }
  }
}

__global__ __launch_bounds__(kVerNT) void verify_sums_kernel(VerArgs A) {
  __shared__ double part[kVerNT / 64][2];
  const int b = blockIdx.y, span = blockIdx.x;
  const VerRow r = verify_row(A.L, b);
  const int v0 = span * kVerSpan + threadIdx.x * kVerPer;
  double2 s = make_double2(0, 0);
  if (v0 < A.L.vocab) {
    float p[kVerPer], q[kVerPer];
    ver_load(r, v0, A.L.vocab, p, q);
#pragma unroll
    for (int i = 0; i < kVerPer; i++) {
      const double2 w = ver_weight(r, p[i], q[i], v0 + i);
      s.x += w.x;
      s.y += w.y;
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    s.x += __shfl_xor(s.x, m);
    s.y += __shfl_xor(s.y, m);
  }
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6][0] = s.x;
    part[threadIdx.x >> 6][1] = s.y;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double t = 0;
    for (int w = 0; w < kVerNT / 64; w++) t += part[w][threadIdx.x];
    A.sums[((int64_t)b * A.spans + span) * 2 + threadIdx.x] = t;
  }
}

// Inclusive sums over the workgroup's threads; *total gets the whole.
__device__ __forceinline__ double ver_scan(double x, double* lds, double* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  __syncthreads();  // lds may still be read from the scan before
  if (lane == 63) lds[w] = x;
  __syncthreads();
  double before = 0, all = 0;
  for (int i = 0; i < kVerNT / 64; i++) {
    if (i < w) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return before + x;
}

__global__ __launch_bounds__(kVerNT) void verify_draw_kernel(VerArgs A) {
  __shared__ double lds[kVerNT / 64];
  __shared__ int first, last;
  const VerifyLaunch& L = A.L;
  const int b = blockIdx.x, t = threadIdx.x;
  VerRow r = verify_row(L, b);
  const double* sums = A.sums + (int64_t)b * A.spans * 2;
  // the whole sums, in span order by threads; of the residual, else of the target
  double all[2];
  for (int k = 0; k < 2; k++) {
    double s = 0;
    for (int i = t; i < A.spans; i += kVerNT) s += sums[2 * i + k];
    ver_scan(s, lds, &all[k]);
  }
  const int which = all[0] > 0.0 ? 0 : 1;
  if (which) r.q = nullptr, r.without = -1;
  const double point = (double)L.uniforms[(int64_t)b * (L.n_new + 1) + L.n_new] * all[which];
  // the first span whose cumulative sum is above the point, else the last with any weight
  double base = 0;
  if (t == 0) first = A.spans, last = -1;
  int span = -1;
  double before = 0;
  for (int i0 = 0; i0 < A.spans; i0 += kVerNT) {
    const int i = i0 + t;
    const double x = i < A.spans ? sums[2 * i + which] : 0.0;
    double total;
    const double c = ver_scan(x, lds, &total);  // its barriers order first and last too
    if (i < A.spans && base + c > point) atomicMin(&first, i);
    if (x > 0.0) atomicMax(&last, i);
    __syncthreads();
    const int f = first;
    if (f < A.spans) {  // the sum before it: from the thread that holds it
      if (i == f) lds[0] = base + (c - x);
      __syncthreads();
      span = f;
      before = lds[0];
      break;
    }
    base += total;
  }
  __syncthreads();
  const bool past = span < 0;
  if (past) span = last;
  int token = -1;
  if (span >= 0) {
    __syncthreads();
    if (t == 0) first = kVerSpan, last = -1;
    const int v0 = span * kVerSpan + t * kVerPer;
    double w[kVerPer], s = 0;
    if (v0 < L.vocab) {
      float p[kVerPer], q[kVerPer];
      ver_load(r, v0, L.vocab, p, q);
#pragma unroll
      for (int i = 0; i < kVerPer; i++) w[i] = which ? ver_weight(r, p[i], q[i], v0 + i).y : ver_weight(r, p[i], q[i], v0 + i).x;
    } else {
#pragma unroll
      for (int i = 0; i < kVerPer; i++) w[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < kVerPer; i++) s += w[i];
    double total;
    double c = before + (ver_scan(s, lds, &total) - s);
    int above = kVerSpan, weight = -1;
#pragma unroll
    for (int i = 0; i < kVerPer; i++) {
      c += w[i];
      if (w[i] > 0.0) {
        weight = t * kVerPer + i;
        if (!past && c > point && above == kVerSpan) above = t * kVerPer + i;
      }
    }
    if (above < kVerSpan) atomicMin(&first, above);
    if (weight >= 0) atomicMax(&last, weight);
    __syncthreads();
    token = span * kVerSpan + (first < kVerSpan ? first : last);
  }
  if (t == 0) L.accepted[b] = r.count;
  for (int j = t; j <= L.n_new; j += kVerNT)
    L.tokens[(int64_t)b * (L.n_new + 1) + j] =
        j < r.count ? L.drafted[(int64_t)b * L.n_new + j] : (j == r.count ? token : -1);
}

}  // namespace

size_t verify_workspace(size_t seqs, size_t vocab) {
  return seqs * ((vocab + kVerSpan - 1) / kVerSpan) * 2 * sizeof(double);
}

hipError_t launch_verify(const VerifyLaunch& L) {
  VerArgs A{L, (double*)L.workspace, (L.vocab + kVerSpan - 1) / kVerSpan};
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
    P.sums += (int64_t)b0 * A.spans * 2;
    hipLaunchKernelGGL(verify_sums_kernel, dim3(A.spans, n), dim3(kVerNT), 0, L.stream, P);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(n), dim3(kVerNT), 0, L.stream, P);
  }
  return hipGetLastError();
}

}  // namespace nrq
