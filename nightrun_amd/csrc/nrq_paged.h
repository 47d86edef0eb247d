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
// A unit's keys and values are read once for all its rows, and that read bounds the kernel where
// there is enough of it: 196,608 positions of two sequences (8 KV heads of 128, f16, 805 MB)
// take 140 to 147 us, 5.5 to 5.75 TB/s, as fast as the card reads at all; 48 sequences of up to 6000 (603 MB)
// 127 us, 4.8 TB/s. 13 sequences under a window of 4096 (178 MB) take 43 us for one new token, 49 for four (16 rows of f32
// queries, one row tile) and 55 for five (20 rows in two); with 16-bit queries 42, 47 and 53. A workgroup has five or six tiles
// of them, so that the chain before the first (length, page, queries, keys) and the join weigh most: the waves
// wait for memory 59% of their time, the matrix units work 8% of theirs. One
// sequence of 1000 positions takes 10 us: two launches and the chain of length, page, key and value.
//
// Per tile each of the four waves takes 32 positions of keys and values straight from
// memory into registers; only the queries' pieces and the join of the waves pass through LDS:
//   S^T = K Q^T on 16x16x32 matrix instructions: lane l holds 16 bytes of row l % 16 of K;
//   O^T += V^T P^T: S^T leaves lane l with the weights of query l % 16 at
//   positions 4 (l / 16) + i of both halves of the tile, which is the order in
//   which P^T wants them if V^T takes its positions in the same order. Lane l reads
//   hd / 16 dimensions of those eight positions and turns the 8 x hd / 16 block around.
// The cache's 16-bit values go into the matrix instructions as they are. f32
// queries go in as sums of 16-bit pieces (scaled by a power of two so that none
// is lost in subnormals), and so do the f32 weights: three bf16 pieces are an f32 value, two f16 pieces are within
// 2^-23 of it (or 2^-37 of the largest). With two bf16 pieces, 2^-17, outputs that cancel would show it; the third takes
// 48 sequences of up to 6000 from 127.0 us to 127.6, thirteen of 9000 by five tokens from 68.4 to 71.1 (bf16).
#include "nrq_page.h"
#include "nrq_serve_launch.h"

namespace nrq {

constexpr int kPaNT = 256;        // threads: four waves
constexpr int kTile = kPagedTile;  // positions of a tile, 32 a wave
constexpr int kPaMaxWgs = 768;
constexpr float kLog2e = 1.44269504088896341f;

struct PaArgs {
  PagedAttnLaunch L;
  int group, rows;      // rows: n_new * group
  int per, row_tiles;   // rows of a unit at most (16 NT), units of a KV head
  int units_per_seq;
  int wgs;
  int slots;            // rows of a unit that there are: min(rows, per)
  int wide_q;           // q in 16-byte loads
  float* part_o;        // [2 * wgs][slots][hd]
  float2* part_ml;      // [2 * wgs][slots]: maximum (log2 units), sum
  int4* share;          // [units]: first and last workgroup, rows
};

inline int pa_per(int hd, size_t rows) { return hd <= 128 && rows > 16 ? 32 : 16; }

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ SeqSpan pa_seq(const PagedAttnLaunch& L, int b) {
  return seq_span(L.lens[b], L.counts ? L.counts[b] : L.n_new, L.n_new, (int64_t)L.table.width * L.kv.page_size,
                  L.window, kTile);
}

// All tiles of the line; the sequence whose tiles hold tile `g(total)`, and its first tile's place.
// Each wave sums and scans the lengths for itself; up to 64 of them are read once.
struct PaLine {
  int total, wgs, at, b, first;
};
__device__ __forceinline__ PaLine pa_line(const PaArgs& A, int wg) {
  const int lane = threadIdx.x & 63, seqs = A.L.table.seqs;
  const int mine = lane < seqs ? pa_seq(A.L, lane).tiles * A.units_per_seq : 0;
  int t = mine;
  for (int b = lane + 64; b < seqs; b += 64) t += pa_seq(A.L, b).tiles * A.units_per_seq;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) t += __shfl_xor(t, m);
  PaLine p;
  p.total = __builtin_amdgcn_readfirstlane(t);
  p.wgs = min(A.wgs, p.total);
  p.at = wg < p.wgs ? line_start(wg, p.total, p.wgs) : p.total;
  int base = 0;
  for (int b0 = 0; b0 < seqs; b0 += 64) {
    const int own = b0 == 0 ? mine : (b0 + lane < seqs ? pa_seq(A.L, b0 + lane).tiles * A.units_per_seq : 0);
    int sum = own;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int y = __shfl_up(sum, m);
      if (lane >= m) sum += y;
    }
    const unsigned long long over = __ballot(base + sum > p.at);
    if (over) {
      const int k = __ffsll(over) - 1;
      p.first = base + __builtin_amdgcn_readlane(sum - own, k);
      p.b = b0 + k;
      return p;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  p.b = seqs, p.first = base;
  return p;
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
  static constexpr int kId = kF16;
  static constexpr int kPieces = 2;  // of an f32 value
  static constexpr uint32_t kExp = 0x7c00u;
  static constexpr float kOffset = 12.0f;  // weights up to 2^12: pieces down to 2^-36 of the largest
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct PaType<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr int kId = kBF16;
  static constexpr int kPieces = 3;
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr float kOffset = 0.0f;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Eight consecutive values of a query.
template <typename Q>
__device__ __forceinline__ void pa_load8(const Q* p, bool wide, float* f) {
  constexpr int V = 16 / sizeof(Q);
  struct alignas(16) Vec {
    Q v[V];
  };
  if (wide) {
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      const Vec a = *(const Vec*)(p + i);
#pragma unroll
      for (int j = 0; j < V; j++) f[i + j] = (float)a.v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)p[i];
  }
}

template <typename Q, int KS>
__device__ __forceinline__ void pa_load_q(const void* q, int64_t at, bool wide, float (*f)[8]) {
#pragma unroll
  for (int s = 0; s < KS; s++) pa_load8((const Q*)q + at + 32 * s, wide, f[s]);
}

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

__device__ __forceinline__ uint32_t pa_place(const PagedAttnLaunch& L, const int* pages, int t, int begin, int end) {
  if (t < begin || t >= end) return kNoPlace;
  return page_place(pages, L.table.width, L.kv.page_size, L.kv.n_pages, L.kv.page_stride8, L.kv.pos_stride8, t);
}

// A wave's 32 positions of a tile in registers: what lane l holds is said above.
template <int HD>
struct PaTile {
  static constexpr int KS = HD / 32, DV = HD / 16;
  u32x4 k[2][KS];
  uint32_t v[8][DV / 2];

  // here: lane p % 32 has the place of position p. Positions without one read the pool's first
  // (any; their scores are masked, their values cleared): no load is conditional.
  __device__ __forceinline__ void load_k(const uint16_t* pool, uint32_t here, int c, int g) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint32_t a = __shfl((int)here, 16 * u + c);
      const uint16_t* p = pool + (uint64_t)a * 8 + 8 * g;
#pragma unroll
      for (int s = 0; s < KS; s++) k[u][s] = *(const u32x4*)(p + 32 * s);
    }
  }
  __device__ __forceinline__ void load_v(const uint16_t* pool, uint32_t here, int c, int g) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t a = __shfl((int)here, (j < 4 ? 0 : 16) + 4 * g + (j & 3));
      const uint16_t* p = pool + (uint64_t)a * 8 + DV * c;
      if constexpr (DV % 8 == 0) {
#pragma unroll
        for (int d = 0; d < DV / 8; d++) {
          const u32x4 x = *(const u32x4*)(p + 8 * d);
#pragma unroll
          for (int i = 0; i < 4; i++) v[j][4 * d + i] = x[i];
        }
      } else if constexpr (DV == 4) {
        const u32x2 x = *(const u32x2*)p;
        v[j][0] = x[0], v[j][1] = x[1];
      } else {
#pragma unroll
        for (int d = 0; d < DV / 2; d++) v[j][d] = ((const uint32_t*)p)[d];
      }
    }
  }
  __device__ __forceinline__ void clear_v(uint32_t live, int g) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const bool on = live >> ((j < 4 ? 0 : 16) + 4 * g + (j & 3)) & 1;
#pragma unroll
      for (int d = 0; d < DV / 2; d++) v[j][d] = on ? v[j][d] : 0u;
    }
  }
};

// Workgroups a CU holds: registers for the tile, the accumulators and the queries.
constexpr int pa_resident(int hd, int nt) { return hd > 128 ? 1 : (nt == 2 || hd > 96 ? 2 : 3); }

// The same stretch of one wave without matrix instructions, position by position and row by
// row, for values that hold an infinity or a NaN: there the products of weights
// that are 0 (rows that do not see a position) or of the pieces of a weight would give
// NaN. Dimension lane + 64 e is the lane's.
template <typename T, int HD>
__device__ __forceinline__ void pa_plain(const PaArgs& A, int b, int head, int row0, int rows, int p0, int stop, int len,
                                      int n, float* ex_o, float (*ex_ml)[2], int os) {
  constexpr int E = (HD + 63) / 64;
  const PagedAttnLaunch& L = A.L;
  const int lane = threadIdx.x & 63;
  const int* pages = L.table.pages + b * L.table.stride;
  for (int r = 0; r < rows; r++) {
    const int rr = row0 + r, tok = rr / A.group, hi = len - n + tok;
    const int lo = L.window > 0 ? max(0, hi - L.window + 1) : 0;
    const int64_t qa = b * L.qb + tok * L.qt + (head * A.group + rr - tok * A.group) * L.qh;
    float q[E], o[E], m = -INFINITY, l = 0;
    for (int e = 0; e < E; e++) {
      const int d = 64 * e + lane;
      o[e] = 0;
      q[e] = 0;
      if (d < HD)
        q[e] = L.dtype == kF32   ? ((const float*)L.q)[qa + d]
               : L.dtype == kF16 ? (float)((const _Float16*)L.q)[qa + d]
                                 : (float)((const __bf16*)L.q)[qa + d];
    }
    for (int t0 = p0; t0 < stop; t0 += kTile)
      for (int t = max(t0, lo); t < min(t0 + 32, hi + 1); t++) {
        const uint32_t place = pa_place(L, pages, t, lo, min(len, hi + 1));
        if (place == kNoPlace) continue;
        const int64_t at = (int64_t)place * 8 + head * L.kv.head_stride;
        float s = 0;
        for (int e = 0; e < E; e++)
          if (64 * e + lane < HD) s = fmaf((float)((const T*)L.kv.k)[at + 64 * e + lane], q[e], s);
        for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
        s *= L.scale * kLog2e;
        const float mn = fmaxf(m, s), by = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
        const float p = __builtin_amdgcn_exp2f(s - (mn == -INFINITY ? 0.0f : mn) + PaType<T>::kOffset);
        l = l * by + p;
        for (int e = 0; e < E; e++)
          if (64 * e + lane < HD) o[e] = o[e] * by + p * (float)((const T*)L.kv.v)[at + 64 * e + lane];
        m = mn;
      }
    for (int e = 0; e < E; e++)
      if (64 * e + lane < HD) ex_o[(64 * e + lane) * os + r] = o[e];
    if (lane == 0) ex_ml[r][0] = m, ex_ml[r][1] = l;
  }
}

// T: the cache's type; HD; NT: groups of 16 rows; NQ: pieces of a query.
template <typename T, int HD, int NT, int NQ>
__global__ __launch_bounds__(kPaNT, pa_resident(HD, NT)) void paged_kernel(PaArgs A) {
  typedef typename PaType<T>::v8 v8;
  constexpr int NP = PaType<T>::kPieces;  // of a weight
  constexpr int KS = HD / 32;  // steps of K
  constexpr int DV = HD / 16;  // dimensions of a lane's values
  constexpr int OS = 16 * NT + 1;  // row stride of the exchange: odd
  __shared__ float ex_ml[4][NT * 16][2], unit_log2[NT * 16];
  // the queries' pieces while a stretch runs, the waves' results behind it
  constexpr int QB = NQ * NT * KS * 64 * 16, OB = 4 * HD * OS * 4;
  __shared__ __align__(16) uint8_t shared[QB > OB ? QB : OB];
  float (*ex_o)[HD * OS] = (float (*)[HD * OS])shared;
  u32x4* qs = (u32x4*)shared;  // [k][n][s][lane]
  const PagedAttnLaunch& L = A.L;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;

  const PaLine line = pa_line(A, blockIdx.x);
  const int total = line.total, wgs = line.wgs;
  if ((int)blockIdx.x >= wgs) return;
  int at = line.at, first = line.first, b = line.b;
  const int stop = line_start(blockIdx.x + 1, total, wgs);
  while (at < stop) {
    const SeqSpan sq = pa_seq(L, b);
    const int unit = (at - first) / sq.tiles;
    const int t_begin = at - first - unit * sq.tiles;
    const int t_end = min(sq.tiles, t_begin + (stop - at));
    const int head = unit / A.row_tiles, rt = unit - head * A.row_tiles;
    const int row0 = rt * 16 * NT, rows = min(16 * NT, sq.n * A.group - row0);
    const bool whole = t_begin == 0 && t_end == sq.tiles;
    if (t_begin == 0 && threadIdx.x == 0)
      A.share[b * A.units_per_seq + unit] =
          make_int4(blockIdx.x, whole ? (int)blockIdx.x : line_owner(at + sq.tiles - 1, total, wgs), rows, 0);
    if (rows > 0) {
      const int first_hi = sq.len - sq.n + row0 / A.group;                // what the unit's first
      const int last_hi = sq.len - sq.n + (row0 + rows - 1) / A.group;    // and last row see
      const int last_lo = L.window > 0 ? max(0, last_hi - L.window + 1) : 0;
      const int begin = L.window > 0 ? max(0, first_hi - L.window + 1) : 0, end = min(sq.len, last_hi + 1);
      const int* pages = L.table.pages + b * L.table.stride;
      const uint16_t* kp = L.kv.k + head * L.kv.head_stride;
      const uint16_t* vp = L.kv.v + head * L.kv.head_stride;
      const int pw = sq.start + 32 * w + (lane & 31);  // the lane's position in the first tile
      uint32_t here = pa_place(L, pages, pw + t_begin * kTile, begin, end);
      PaTile<HD> tile;
      uint32_t live = (uint32_t)__ballot(here != kNoPlace), next = kNoPlace, next_live = 0;
      if (live) {  // else the pool may be empty
        tile.load_k(kp, here == kNoPlace ? 0 : here, c, g);
        tile.load_v(vp, here == kNoPlace ? 0 : here, c, g);
      }
      if (t_begin + 1 < t_end) {
        next = pa_place(L, pages, pw + (t_begin + 1) * kTile, begin, end);
        next_live = (uint32_t)__ballot(next != kNoPlace);
      }
      // ---- queries: wave n brings the pieces of group n to LDS, in registers they would cost the
      // workgroups of a CU that hide the loads
      __syncthreads();  // the exchange of the unit before is read
      if (w < NT) {
        const int r = min(row0 + 16 * w + c, sq.n * A.group - 1), tok = r / A.group;
        const int64_t qa = b * L.qb + tok * L.qt + (head * A.group + r - tok * A.group) * L.qh + 8 * g;
        float f[KS][8], unit = L.scale * kLog2e;
        if (NQ == 1)
          pa_load_q<T, KS>(L.q, qa, A.wide_q, f);  // 16 bits either way: the conversions cancel
        else if (L.dtype == kF32)
          pa_load_q<float, KS>(L.q, qa, A.wide_q, f);
        else if (L.dtype == kF16)
          pa_load_q<_Float16, KS>(L.q, qa, A.wide_q, f);
        else
          pa_load_q<__bf16, KS>(L.q, qa, A.wide_q, f);
        if (NQ > 1) {  // the largest magnitude of the row to [2^13, 2^14)
          float big = 0.0f;
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(f[s][i]));
          big = fmaxf(big, __shfl_xor(big, 16));
          big = fmaxf(big, __shfl_xor(big, 32));
          const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253);  // small rows: as if 2^-100
          const float up = __uint_as_float((uint32_t)(267 - e) << 23);
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) f[s][i] *= up;
          unit *= 1.0f / up;
        }
#pragma unroll
        for (int s = 0; s < KS; s++) {
          v8 tmp[NQ];
          pa_split<T, NQ>(f[s], tmp);
#pragma unroll
          for (int k = 0; k < NQ; k++) qs[((k * NT + w) * KS + s) * 64 + lane] = *(u32x4*)&tmp[k];
        }
        if (g == 0) unit_log2[16 * w + c] = unit;
      }
      __syncthreads();
      float to_log2[NT];  // what brings a row's products to log2 units
      int lo[NT], hi[NT];  // what the row sees
#pragma unroll
      for (int n = 0; n < NT; n++) {
        to_log2[n] = unit_log2[16 * n + c];
        hi[n] = sq.len - sq.n + min(row0 + 16 * n + c, sq.n * A.group - 1) / A.group;
        lo[n] = L.window > 0 ? max(0, hi[n] - L.window + 1) : 0;
      }

      float m[NT], l[NT];
      f32x4 acc[NT][DV];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DV; d++) acc[n][d] = f32x4{0, 0, 0, 0};
      }
      int p0 = sq.start + t_begin * kTile + 32 * w;
      for (int t = t_begin; t < t_end; t++, p0 += kTile) {
        uint32_t after = kNoPlace;
        if (t + 2 < t_end) after = pa_place(L, pages, pw + (t + 2) * kTile, begin, end);
        // ---- scores: 8 positions for query c of each group
        f32x4 x[NT][2];
        if (live) {
          asm volatile("" ::: "memory");  // the queries stay in LDS
#pragma unroll
          for (int n = 0; n < NT; n++) {
            x[n][0] = x[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = NQ - 1; k >= 0; k--)
#pragma unroll
              for (int s = 0; s < KS; s++) {
                const u32x4 q = qs[((k * NT + n) * KS + s) * 64 + lane];
                x[n][0] = PaType<T>::mfma(*(v8*)&tile.k[0][s], *(v8*)&q, x[n][0]);
                x[n][1] = PaType<T>::mfma(*(v8*)&tile.k[1][s], *(v8*)&q, x[n][1]);
              }
          }
        }
        const uint32_t ahead = next == kNoPlace ? 0 : next;
        if (next_live) tile.load_k(kp, ahead, c, g);
        if (live) {
          const bool inside = live == 0xffffffffu && p0 + 31 <= first_hi && p0 >= last_lo;
          v8 pp[NT][NP];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] = x[n][i >> 2][i & 3] * to_log2[n];
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
            pa_split<T, NP>(p, pp[n]);
          }
          if (live != 0xffffffffu) tile.clear_v(live, g);
          // ---- O^T += V^T P^T
#pragma unroll
          for (int d = 0; d < DV; d++) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; j++)  // a pair of positions of one dimension
              a[j] = __builtin_amdgcn_perm(tile.v[2 * j + 1][d / 2], tile.v[2 * j][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int k = NP - 1; k >= 0; k--) acc[n][d] = PaType<T>::mfma(*(v8*)&a, pp[n][k], acc[n][d]);
          }
        }
        if (next_live) tile.load_v(vp, ahead, c, g);
        live = next_live;
        next = after;
        next_live = (uint32_t)__ballot(next != kNoPlace);
      }
      // ---- the four waves' results together
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
#pragma unroll
        for (int d = 0; d < DV; d++)
          sum += (acc[n][d][0] * 0.0f + acc[n][d][1] * 0.0f) + (acc[n][d][2] * 0.0f + acc[n][d][3] * 0.0f);
      }
      __syncthreads();  // the queries are read
      if (__any(sum != sum)) {
        pa_plain<T, HD>(A, b, head, row0, rows, sq.start + t_begin * kTile + 32 * w, sq.start + t_end * kTile, sq.len,
                        sq.n, ex_o[w], ex_ml[w], OS);
      } else {
#pragma unroll
        for (int n = 0; n < NT; n++)
          if (16 * n + c < rows) {
            if (g == 0) {
              ex_ml[w][16 * n + c][0] = m[n];
              ex_ml[w][16 * n + c][1] = l[n];
            }
#pragma unroll
            for (int d = 0; d < DV; d++)
#pragma unroll
              for (int i = 0; i < 4; i++) ex_o[w][((4 * g + i) * DV + d) * OS + 16 * n + c] = acc[n][d][i];
          }
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
          const float by = __builtin_amdgcn_exp2f(ex_ml[k][r][0] - ref);
          if (by > 0.0f || ref != ref) o += ex_o[k][d * OS + r] * by;  // a wave that saw nothing, or nothing of weight
          ll += ex_ml[k][r][1] * by;
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
    if (at == first + sq.tiles * A.units_per_seq) {
      first = at;
      b++;
    }
  }
}

// The stretches of one row of a unit that several workgroups shared, in order: four waves take
// every fourth of them, then add up.
template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PaArgs A) {
  constexpr int E = (HD + 63) / 64;  // dimensions of a lane: lane + 64 e
  __shared__ float ex_o[4][64 * E], ex_l[4];
  const PagedAttnLaunch& L = A.L;
  const int u = blockIdx.x, b = u / A.units_per_seq, unit = u - b * A.units_per_seq;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int4 share = A.share[u];
  const int r = blockIdx.y, w0 = share.x, n = share.y - w0 + 1;
  if (n < 2 || r >= share.z) return;
  const int head = unit / A.row_tiles, rr = (unit - head * A.row_tiles) * A.per + r;
  auto slot = [&](int k) { return (int64_t)(2 * (w0 + k) + (k == 0 ? 1 : 0)) * A.slots + r; };
  // the maximum over all stretches, then their sums; a lane keeps the first 64's
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (lane < n) ml = A.part_ml[slot(lane)];
  float mm = ml.x;
  for (int k = lane + 64; k < n; k += 64) mm = fmaxf(mm, A.part_ml[slot(k)].x);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) mm = fmaxf(mm, __shfl_xor(mm, m));
  const float ref = mm == -INFINITY ? 0.0f : mm;
  const float mine = __builtin_amdgcn_exp2f(ml.x - ref);
  float o[E], l = 0;
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = 0;
#pragma unroll 8
  for (int k = w; k < min(n, 64); k += 4) {
    const float by = __shfl(mine, k);
    l += __shfl(ml.y, k) * by;
    const int64_t s = slot(k);
#pragma unroll
    for (int e = 0; e < E; e++)
      if (64 * e + lane < HD) o[e] += A.part_o[s * HD + 64 * e + lane] * by;
  }
#pragma unroll 4
  for (int k = 64 + w; k < n; k += 4) {
    const int64_t s = slot(k);
    const float2 x = A.part_ml[s];
    const float by = __builtin_amdgcn_exp2f(x.x - ref);
    l += x.y * by;
#pragma unroll
    for (int e = 0; e < E; e++)
      if (64 * e + lane < HD) o[e] += A.part_o[s * HD + 64 * e + lane] * by;
  }
#pragma unroll
  for (int e = 0; e < E; e++) ex_o[w][64 * e + lane] = o[e];
  if (lane == 0) ex_l[w] = l;
  __syncthreads();
  l = ((ex_l[0] + ex_l[1]) + (ex_l[2] + ex_l[3]));
  const int tok = rr / A.group, h = head * A.group + rr - tok * A.group;
  const bool none = mm == -INFINITY && l == 0.0f;
  for (int d = threadIdx.x; d < HD; d += 256) {
    const float x = (ex_o[0][d] + ex_o[1][d]) + (ex_o[2][d] + ex_o[3][d]);
    pa_store(L.out, L.dtype, b * L.ob + tok * L.ot + h * L.oh + d, none ? 0.0f : x / l);
  }
  if (L.lse && threadIdx.x == 0)
    L.lse[((int64_t)b * L.n_new + tok) * L.heads + h] =
        none ? -INFINITY : (mm - PaType<T>::kOffset + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int HD, int NT, int NQ>
hipError_t pa_launch(PaArgs& A) {
  const int64_t units = (int64_t)A.units_per_seq * A.L.table.seqs;
  const int64_t tiles = ((int64_t)A.L.table.width * A.L.kv.page_size + kTile - 1) / kTile;
  const int64_t most = units * (tiles > 0 ? tiles : 1), fill = 256 * pa_resident(HD, NT);
  static_assert(256 * pa_resident(HD, NT) <= kPaMaxWgs, "workspace");
  A.wgs = (int)(most < fill ? most : fill);
  A.part_o = (float*)A.L.workspace;
  A.part_ml = (float2*)(A.part_o + (size_t)2 * A.wgs * A.slots * HD);
  A.share = (int4*)(((uintptr_t)(A.part_ml + (size_t)2 * A.wgs * A.slots) + 15) & ~(uintptr_t)15);
  hipLaunchKernelGGL((paged_kernel<T, HD, NT, NQ>), dim3(A.wgs), dim3(kPaNT), 0, A.L.stream, A);
  if (tiles > 1)
    hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3((unsigned)units, A.slots), dim3(256), 0, A.L.stream, A);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t pa_launch_hd(const PagedAttnLaunch& L) {
  constexpr int kMany = PaType<T>::kPieces;
  PaArgs A;
  A.L = L;
  A.group = L.heads / L.kv.n_kv;
  A.rows = L.n_new * A.group;
  A.per = pa_per(HD, A.rows);
  A.row_tiles = (A.rows + A.per - 1) / A.per;
  A.units_per_seq = L.kv.n_kv * A.row_tiles;
  A.slots = A.rows < A.per ? A.rows : A.per;
  const int v = L.dtype == kF32 ? 4 : 8;
  A.wide_q = ((uintptr_t)L.q & 15) == 0 && L.qb % v == 0 && L.qt % v == 0 && L.qh % v == 0;
  const bool same = L.dtype == PaType<T>::kId;
  if constexpr (HD <= 128)
    if (A.per == 32) return same ? pa_launch<T, HD, 2, 1>(A) : pa_launch<T, HD, 2, kMany>(A);
  return same ? pa_launch<T, HD, 1, 1>(A) : pa_launch<T, HD, 1, kMany>(A);
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
