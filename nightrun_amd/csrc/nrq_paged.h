// Attention of new tokens over a paged cache (include/nrq_serve.h,
// nrq_dev_paged_attention): the kernels, instantiated per cache type in
// nrq_paged_f16.hip and nrq_paged_bf16.hip.
//
// A unit is one sequence, one KV head and up to 16 NT of its rows (new tokens x
// query heads of the group); its positions are cut into tiles of kTile. All
// tiles of all units form one line, and every workgroup takes an equal stretch of
// it, so ragged lengths load the card evenly and one long sequence fills it. Within
// a unit the running maximum and sum of the softmax are kept (weights 2^(s - m),
// s in units of log2); a stretch that holds a whole unit writes the output, the
// others write (m, l, o) to the workspace, which a second launch joins in order.
//
// Per tile each of the four waves takes 32 positions straight from memory into
// registers, nothing passes through LDS:
//   S^T = K Q^T on 16x16x32 matrix instructions: lane l holds 16 bytes of row l % 16 of K;
//   O^T += V^T P^T: S^T leaves lane l with the weights of query l % 16 at
//   positions 4 (l / 16) + i of both halves of the tile, which is the order in
//   which P^T wants them if V^T takes its positions in the same order. Lane l reads
//   hd / 16 dimensions of those eight positions and turns the 8 x hd / 16 block around.
// The cache's 16-bit values go into the matrix instructions as they are. f32
// queries go in as sums of 16-bit pieces (scaled by a power of two so that none
// is lost in subnormals), and so do the f32 weights: two f16 pieces keep 22 bits,
// three bf16 pieces 24, two bf16 pieces 16 (for 16-bit outputs, whose own
// rounding is 2^-9). The kernel waits on memory, the extra products are free.
#include "nrq_page.h"
#include "nrq_serve_launch.h"

namespace nrq {

constexpr int kPaNT = 256;        // threads: four waves
constexpr int kTile = 128;        // positions of a tile, 32 a wave
constexpr int kPaMaxWgs = 1024;   // four workgroups on each of 256 CUs
constexpr float kLog2e = 1.44269504088896341f;

struct PaArgs {
  PagedAttnLaunch L;
  int group, rows;      // rows: n_new * group
  int per, row_tiles;   // rows of a unit at most (16 NT), units of a KV head
  int units_per_seq;
  int wgs;
  int slots;            // rows of a unit that there are: min(rows, per)
  float* part_o;        // [2 * wgs][slots][hd]
  float2* part_ml;      // [2 * wgs][slots]: maximum (log2 units), sum
};

inline int pa_per(int hd, size_t rows) { return hd <= 128 && rows > 16 ? 32 : 16; }

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ SeqSpan pa_seq(const PagedAttnLaunch& L, int b) {
  return seq_span(L.lens[b], L.counts ? L.counts[b] : L.n_new, L.n_new, (int64_t)L.table.width * L.kv.page_size,
                  L.window, kTile);
}

// All tiles of a sequence's units, and of the sequences before it: a wave's own
// scan over the lengths.
__device__ __forceinline__ int64_t pa_total(const PaArgs& A) {
  const int lane = threadIdx.x & 63;
  int64_t t = 0;
  for (int b = lane; b < A.L.table.seqs; b += 64) t += pa_seq(A.L, b).tiles;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) t += __shfl_xor(t, m);
  return t * A.units_per_seq;
}

// The sequence whose tiles hold tile g of the line, and its first tile's place.
__device__ __forceinline__ int pa_find(const PaArgs& A, int64_t g, int64_t* first) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0;
  for (int b0 = 0; b0 < A.L.table.seqs; b0 += 64) {
    const int b = b0 + lane;
    int64_t own = b < A.L.table.seqs ? (int64_t)pa_seq(A.L, b).tiles * A.units_per_seq : 0, sum = own;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t y = __shfl_up(sum, m);
      if (lane >= m) sum += y;
    }
    const unsigned long long over = __ballot(base + sum > g);
    if (over) {
      const int at = __ffsll(over) - 1;
      *first = base + __shfl(sum, at) - __shfl(own, at);
      return b0 + at;
    }
    base += __shfl(sum, 63);
  }
  *first = base;
  return A.L.table.seqs;
}

__device__ __forceinline__ float pa_load_q(const void* q, int dtype, int64_t at) {
  if (dtype == kF32) return ((const float*)q)[at];
  return dtype == kF16 ? (float)((const _Float16*)q)[at] : (float)((const __bf16*)q)[at];
}

__device__ __forceinline__ void pa_store(void* o, int dtype, int64_t at, float v) {
  if (dtype == kF32)
    ((float*)o)[at] = v;
  else if (dtype == kF16)
    ((_Float16*)o)[at] = (_Float16)v;
  else
    ((__bf16*)o)[at] = (__bf16)v;
}

template <typename T>
struct PaType;
template <>
struct PaType<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExp = 0x7c00u;
  static constexpr float kOffset = 12.0f;  // weights up to 2^12: pieces down to 2^-36 of the largest
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct PaType<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr float kOffset = 0.0f;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Pieces of eight f32 values, each the rest of the ones before it.
template <typename T, int N>
__device__ __forceinline__ void pa_split(const float* f, typename PaType<T>::v8* out) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = f[i];
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const T h = (T)r[i];
      out[k][i] = h;
      r[i] -= (float)h;
    }
}

__device__ __forceinline__ int64_t pa_place(const PagedAttnLaunch& L, const int* pages, int t, int begin, int end) {
  if (t < begin || t >= end) return -1;
  return page_place(pages, L.table.width, L.kv.page_size, L.kv.n_pages, L.kv.page_stride, L.kv.pos_stride, t);
}

// T: the cache's type; HD; NT: groups of 16 rows; NQ, NP: pieces of a query and of a weight.
template <typename T, int HD, int NT, int NQ, int NP>
__global__ __launch_bounds__(kPaNT) void paged_kernel(PaArgs A) {
  typedef typename PaType<T>::v8 v8;
  constexpr int KS = HD / 32;  // steps of K
  constexpr int DV = HD / 16;  // dimensions of a lane's values
  constexpr int OS = 16 * NT + 1;  // row stride of the exchange: odd
  __shared__ float ex_ml[4][NT * 16][2];
  __shared__ float ex_o[4][HD * OS];
  const PagedAttnLaunch& L = A.L;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;

  const int64_t total = pa_total(A);
  const int64_t wgs = min<int64_t>(A.wgs, total);
  if (blockIdx.x >= wgs) return;
  int64_t at = line_start(blockIdx.x, total, wgs);
  const int64_t stop = line_start((int64_t)blockIdx.x + 1, total, wgs);
  int64_t first;
  int b = pa_find(A, at, &first);
  while (at < stop) {
    const SeqSpan sq = pa_seq(L, b);
    const int unit = (int)((at - first) / sq.tiles);
    const int t_begin = (int)(at - first - (int64_t)unit * sq.tiles);
    const int t_end = (int)min<int64_t>(sq.tiles, t_begin + (stop - at));
    const int head = unit / A.row_tiles, rt = unit - head * A.row_tiles;
    const int row0 = rt * 16 * NT, rows = min(16 * NT, sq.n * A.group - row0);
    const bool whole = t_begin == 0 && t_end == sq.tiles;
    if (rows > 0) {
      // ---- queries, and what each row sees
      v8 q[NQ][NT][KS];
      float to_log2[NT];  // what brings a row's products to log2 units
      int lo[NT], hi[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int r = min(row0 + 16 * n + c, sq.n * A.group - 1), tok = r / A.group;
        hi[n] = sq.len - sq.n + tok;
        lo[n] = L.window > 0 ? max(0, hi[n] - L.window + 1) : 0;
        const int64_t qa = b * L.qb + tok * L.qt + (head * A.group + r - tok * A.group) * L.qh;
        float f[KS][8], big = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            f[s][i] = pa_load_q(L.q, L.dtype, qa + 32 * s + 8 * g + i);
            big = fmaxf(big, fabsf(f[s][i]));
          }
        to_log2[n] = L.scale * kLog2e;
        if (NQ > 1) {  // the largest magnitude of the row to [2^13, 2^14)
          big = fmaxf(big, __shfl_xor(big, 16));
          big = fmaxf(big, __shfl_xor(big, 32));
          const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253);  // small rows: as if 2^-100
          const float up = __uint_as_float((uint32_t)(267 - e) << 23);
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) f[s][i] *= up;
          to_log2[n] *= 1.0f / up;
        }
#pragma unroll
        for (int s = 0; s < KS; s++) {
          v8 tmp[NQ];
          pa_split<T, NQ>(f[s], tmp);
#pragma unroll
          for (int k = 0; k < NQ; k++) q[k][n][s] = tmp[k];
        }
      }
      const int first_row_hi = sq.len - sq.n + row0 / A.group;                 // of the unit's rows the
      const int last_row_hi = sq.len - sq.n + (row0 + rows - 1) / A.group;     // nearest and farthest ends
      const int last_row_lo = L.window > 0 ? max(0, last_row_hi - L.window + 1) : 0;
      // positions that any of them sees
      const int begin = L.window > 0 ? max(0, first_row_hi - L.window + 1) : 0, end = min(sq.len, last_row_hi + 1);

      const int* pages = L.table.pages + b * L.table.stride;
      const T* kp = (const T*)L.kv.k + head * L.kv.head_stride;
      const T* vp = (const T*)L.kv.v + head * L.kv.head_stride;

      float m[NT], l[NT];
      f32x4 acc[NT][DV];
      // With an infinity or a NaN among the values the plain sums go wrong: a weight of 0 (a
      // row that does not see the position) or a negative piece of one times infinity is
      // NaN. Such a stretch is done again, `apart`: row by row, each with the values that it sees,
      // and the lower pieces with the finite ones only.
      bool apart = false;
    again:
#pragma unroll
      for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DV; d++) acc[n][d] = f32x4{0, 0, 0, 0};
      }
      int p0 = sq.start + t_begin * kTile + 32 * w;
      int64_t place = pa_place(L, pages, p0 + (lane & 31), begin, end);
      for (int t = t_begin; t < t_end; t++, p0 += kTile) {
        if (p0 >= end) break;
        const int64_t here = place;
        if (t + 1 < t_end) place = pa_place(L, pages, p0 + kTile + (lane & 31), begin, end);
        // ---- loads: 32 positions of K and V
        u32x4 kr[2][KS];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int64_t a = __shfl(here, 16 * u + c);
#pragma unroll
          for (int s = 0; s < KS; s++)
            kr[u][s] = a >= 0 ? *(const u32x4*)(kp + a + 32 * s + 8 * g) : u32x4{0, 0, 0, 0};
        }
        uint32_t vr[8][DV / 2];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int64_t a = __shfl(here, (j < 4 ? 0 : 16) + 4 * g + (j & 3));
#pragma unroll
          for (int d = 0; d < DV / 2; d++) vr[j][d] = 0;
          if (a >= 0) {
            if constexpr (DV % 8 == 0) {
#pragma unroll
              for (int d = 0; d < DV / 8; d++) *(u32x4*)&vr[j][4 * d] = *(const u32x4*)(vp + a + DV * c + 8 * d);
            } else {
              struct alignas(4) Row {
                uint32_t x[DV / 2];
              };
              const Row r = *(const Row*)(vp + a + DV * c);
#pragma unroll
              for (int d = 0; d < DV / 2; d++) vr[j][d] = r.x[d];
            }
          }
        }
        // which of the 32 positions are on a page
        const uint32_t live = (uint32_t)__ballot(here >= 0);
        const bool inside = live == 0xffffffffu && p0 + 31 <= first_row_hi && p0 >= last_row_lo;
#pragma unroll
        for (int n = 0; n < NT; n++) {
          // ---- scores of 8 positions for query c, in log2 units
          float s[8];
#pragma unroll
          for (int u = 0; u < 2; u++) {
            f32x4 x = {0, 0, 0, 0};
#pragma unroll
            for (int k = NQ - 1; k >= 0; k--)
#pragma unroll
              for (int st = 0; st < KS; st++) x = PaType<T>::mfma(*(v8*)&kr[u][st], q[k][n][st], x);
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * u + i] = x[i] * to_log2[n];
          }
          if (!inside) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int o = (i < 4 ? 0 : 16) + 4 * g + (i & 3), p = p0 + o;
              s[i] = p >= lo[n] && p <= hi[n] && (live >> o & 1) ? s[i] : -INFINITY;
            }
          }
          // ---- running maximum and sum
          float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float mn = fmaxf(m[n], top);
          const float ref = mn == -INFINITY ? 0.0f : mn;
          if (__any(mn > m[n])) {
            const float by = __builtin_amdgcn_exp2f(m[n] - ref);
            l[n] *= by;
#pragma unroll
            for (int d = 0; d < DV; d++) acc[n][d] *= by;
            m[n] = mn;
          }
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(s[i] - ref + PaType<T>::kOffset);
            l[n] += p[i];
          }
          v8 pp[NP];
          pa_split<T, NP>(p, pp);
          // ---- O^T += V^T P^T
          if (!apart) {
#pragma unroll
            for (int d = 0; d < DV; d++) {
              u32x4 a;
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const uint32_t x = vr[2 * j][d / 2], y = vr[2 * j + 1][d / 2];
                a[j] = d & 1 ? (x >> 16) | (y & 0xffff0000u) : (x & 0xffffu) | (y << 16);
              }
#pragma unroll
              for (int k = NP - 1; k >= 0; k--) acc[n][d] = PaType<T>::mfma(*(v8*)&a, pp[k], acc[n][d]);
            }
          } else {
            for (int j = 0; j < 8; j++)  // a weight above 0 is not lost in the first piece
              if (p[j] > 0.0f && (float)pp[0][j] == 0.0f) pp[0][j] = (T)6e-8f;
#pragma unroll 1
            for (int only = 0; only < 16; only++) {
              const int l0 = __shfl(lo[n], only), h0 = __shfl(hi[n], only);
#pragma unroll
              for (int d = 0; d < DV; d++) {
                u32x4 a, fin;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  uint32_t h[2];
#pragma unroll
                  for (int i = 0; i < 2; i++) {
                    const int pos = p0 + (j < 2 ? 0 : 16) + 4 * g + (2 * j & 3) + i;
                    h[i] = (d & 1 ? vr[2 * j + i][d / 2] >> 16 : vr[2 * j + i][d / 2]) & 0xffffu;
                    if (pos < l0 || pos > h0) h[i] = 0;
                  }
                  a[j] = h[0] | h[1] << 16;
#pragma unroll
                  for (int i = 0; i < 2; i++)
                    if ((h[i] & PaType<T>::kExp) == PaType<T>::kExp) h[i] = 0;
                  fin[j] = h[0] | h[1] << 16;
                }
                f32x4 x = acc[n][d];
#pragma unroll
                for (int k = NP - 1; k >= 0; k--) x = PaType<T>::mfma(k ? *(v8*)&fin : *(v8*)&a, pp[k], x);
                if (c == only) acc[n][d] = x;
              }
            }
          }
        }
      }
      if (!apart) {
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int d = 0; d < DV; d++) sum += (acc[n][d][0] * 0.0f + acc[n][d][1] * 0.0f) + (acc[n][d][2] * 0.0f + acc[n][d][3] * 0.0f);
        if (__any(sum != sum)) {
          apart = true;
          goto again;
        }
      }

      // ---- the four waves' results together
      __syncthreads();  // the exchange of the unit before is read
#pragma unroll
      for (int n = 0; n < NT; n++) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (g == 0) {
          ex_ml[w][16 * n + c][0] = m[n];
          ex_ml[w][16 * n + c][1] = l[n];
        }
      }
      __syncthreads();
      float* mine = ex_o[w];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float mm = ex_ml[0][16 * n + c][0];
#pragma unroll
        for (int i = 1; i < 4; i++) mm = fmaxf(mm, ex_ml[i][16 * n + c][0]);
        const float by = __builtin_amdgcn_exp2f(m[n] - (mm == -INFINITY ? 0.0f : mm));
#pragma unroll
        for (int d = 0; d < DV; d++)
#pragma unroll
          for (int i = 0; i < 4; i++) mine[((4 * g + i) * DV + d) * OS + 16 * n + c] = acc[n][d][i] * by;
      }
      __syncthreads();
      const int64_t slot = 2 * (int64_t)blockIdx.x + (t_begin == 0 ? 1 : 0);
      for (int i = threadIdx.x; i < rows * HD; i += kPaNT) {
        const int r = i / HD, d = i - r * HD;
        float o = 0, mm = ex_ml[0][r][0], ll = 0;
#pragma unroll
        for (int k = 1; k < 4; k++) mm = fmaxf(mm, ex_ml[k][r][0]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          o += ex_o[k][d * OS + r];
          ll += ex_ml[k][r][1] * __builtin_amdgcn_exp2f(ex_ml[k][r][0] - ref);
        }
        if (!whole) {
          A.part_o[(slot * A.slots + r) * HD + d] = o;
          if (d == 0) A.part_ml[slot * A.slots + r] = make_float2(mm, ll);
        } else {
          const int rr = row0 + r, tok = rr / A.group, h = head * A.group + rr - tok * A.group;
          const bool none = mm == -INFINITY && ll == 0.0f;
          pa_store(L.out, L.dtype, b * L.ob + tok * L.ot + h * L.oh + d, none ? 0.0f : o / ll);
          if (L.lse && d == 0)
            L.lse[((int64_t)b * L.n_new + tok) * L.heads + h] =
                none ? -INFINITY : (mm - PaType<T>::kOffset + log2f(ll)) * 0.69314718055994531f;
        }
      }
    }
    at += t_end - t_begin;
    if (at == first + (int64_t)sq.tiles * A.units_per_seq) {
      first = at;
      b++;
    }
  }
}

// The stretches of one row of a unit that more than one workgroup shared, in order.
template <typename T, int HD>
__global__ __launch_bounds__((HD + 63) / 64 * 64) void paged_join_kernel(PaArgs A) {
  const PagedAttnLaunch& L = A.L;
  const int u = blockIdx.x, b = u / A.units_per_seq, unit = u - b * A.units_per_seq;
  const int lane = threadIdx.x & 63;
  const SeqSpan sq = pa_seq(L, b);
  const int head = unit / A.row_tiles, rt = unit - head * A.row_tiles;
  const int r = blockIdx.y, rr = rt * A.per + r;
  if (rr >= sq.n * A.group) return;
  int64_t before = 0;
  for (int i = lane; i < b; i += 64) before += pa_seq(L, i).tiles;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) before += __shfl_xor(before, m);
  const int64_t total = pa_total(A), wgs = min<int64_t>(A.wgs, total);
  const int64_t g0 = before * A.units_per_seq + (int64_t)unit * sq.tiles, g1 = g0 + sq.tiles;
  const int64_t w0 = line_owner(g0, total, wgs), w1 = line_owner(g1 - 1, total, wgs);
  if (w0 == w1) return;
  const int d = threadIdx.x;
  float mm = -INFINITY;
  for (int64_t k = w0; k <= w1; k++) mm = fmaxf(mm, A.part_ml[(2 * k + (k == w0 ? 1 : 0)) * A.slots + r].x);
  const float ref = mm == -INFINITY ? 0.0f : mm;
  float o = 0, l = 0;
  for (int64_t k = w0; k <= w1; k++) {
    const int64_t slot = (2 * k + (k == w0 ? 1 : 0)) * A.slots + r;
    const float2 ml = A.part_ml[slot];
    const float by = __builtin_amdgcn_exp2f(ml.x - ref);
    l += ml.y * by;
    if (d < HD) o += A.part_o[slot * HD + d] * by;
  }
  const int tok = rr / A.group, h = head * A.group + rr - tok * A.group;
  const bool none = mm == -INFINITY && l == 0.0f;
  if (d < HD) pa_store(L.out, L.dtype, b * L.ob + tok * L.ot + h * L.oh + d, none ? 0.0f : o / l);
  if (L.lse && d == 0)
    L.lse[((int64_t)b * L.n_new + tok) * L.heads + h] =
        none ? -INFINITY : (mm - PaType<T>::kOffset + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int HD, int NT, int NQ, int NP>
hipError_t pa_launch(PaArgs& A, bool join) {
  hipLaunchKernelGGL((paged_kernel<T, HD, NT, NQ, NP>), dim3(A.wgs), dim3(kPaNT), 0, A.L.stream, A);
  if (join)
    hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3(A.units_per_seq * A.L.table.seqs, A.slots),
                       dim3((HD + 63) / 64 * 64), 0, A.L.stream, A);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t pa_launch_hd(const PagedAttnLaunch& L) {
  constexpr int kMany = sizeof(T) == 2 && PaType<T>::kOffset > 0 ? 2 : 3;  // f16: 2 pieces of 11 bits, bf16: 3 of 8
  PaArgs A;
  A.L = L;
  A.group = L.heads / L.kv.n_kv;
  A.rows = L.n_new * A.group;
  A.per = pa_per(HD, A.rows);
  A.row_tiles = (A.rows + A.per - 1) / A.per;
  A.units_per_seq = L.kv.n_kv * A.row_tiles;
  const int64_t units = (int64_t)A.units_per_seq * L.table.seqs;
  const int64_t tiles = ((int64_t)L.table.width * L.kv.page_size + kTile - 1) / kTile;
  A.wgs = (int)(units * (tiles > 0 ? tiles : 1) < kPaMaxWgs ? units * (tiles > 0 ? tiles : 1) : kPaMaxWgs);
  A.slots = A.rows < A.per ? A.rows : A.per;
  A.part_o = (float*)L.workspace;
  A.part_ml = (float2*)(A.part_o + (size_t)2 * A.wgs * A.slots * HD);
  const bool join = tiles > 1;
  const bool same = L.dtype == (PaType<T>::kOffset > 0 ? kF16 : kBF16);
  if constexpr (HD <= 128)
    if (A.per == 32)
      return same ? pa_launch<T, HD, 2, 1, 2>(A, join) : pa_launch<T, HD, 2, kMany, kMany>(A, join);
  return same ? pa_launch<T, HD, 1, 1, 2>(A, join) : pa_launch<T, HD, 1, kMany, kMany>(A, join);
}

template <typename T>
hipError_t pa_launch_type(const PagedAttnLaunch& L) {
  switch (L.kv.hd) {
    case 32: return pa_launch_hd<T, 32>(L);
    case 64: return pa_launch_hd<T, 64>(L);
    case 96: return pa_launch_hd<T, 96>(L);
    case 128: return pa_launch_hd<T, 128>(L);
    default: return pa_launch_hd<T, 256>(L);
  }
}

}  // namespace
}  // namespace nrq
