// Attention of a tree's nodes over a paged cache where a KV head has more than 32 rows (nodes x query heads of the
// group): the kernels, instantiated per cache type in nrq_tree_f16.hip and nrq_tree_bf16.hip. Fewer rows, and what is
// common to both (the line of tiles and its stretches, the softmax, pieces of f32 values, the join), are in nrq_paged.h.
//
// With R rows a position of a KV head costs 4 R head_dim operations for 4 head_dim bytes, R operations a byte: from a hundred
// rows on, as many workgroups as there are groups of 32 rows would read the keys and values from L2 more often
// than it delivers. So a unit is up to 256 rows, and its keys and values pass through LDS once for all of them: stage by
// stage, the next one on its way from memory to registers while one is multiplied.
//
// A wave owns 32 rows, with fewer rows than waves a part of each stage's positions (their results are added up in
// LDS at the end of a stretch). Per 32 positions:
//   S^T = K Q^T on 32x32x16 matrix instructions, queries in registers: lane l gets row l % 32 at positions
//   8 i + 4 (l / 32) + j, which is the order in which P^T goes into the second product,
//   O^T += V^T P^T, with V^T read transposed from LDS (four positions of one dimension a lane).
// Rows of K lie an odd number of 16-byte chunks apart and rows of V 64 bytes past a multiple of 128, so that neither read
// meets a bank twice.
#pragma once

#include "nrq_paged.h"
#include "nrq_tree_launch.h"

namespace nrq {

constexpr int kTaWgs = 256;  // workgroups: one a CU

// Rows of a KV head that nrq_paged.h takes: one unit of its.
inline size_t ta_few(int hd) { return hd <= 128 ? 32 : 16; }

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct TaType;
template <>
struct TaType<_Float16> {
  typedef PaType<_Float16>::v8 v8;
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct TaType<__bf16> {
  typedef PaType<__bf16>::v8 v8;
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Four positions of one dimension: of 16 lanes, lanes 4 r .. 4 r + 3 name 16 consecutive values of row r, lane i gets
// the i-th of each of the four rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 ta_read_tr(const uint8_t* p) {
  typedef __attribute__((address_space(3))) s16x4* lds;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)p));
}

// W waves, WR of them side by side over the rows, TP positions of a stage.
template <int HD, int W, int WR, int TP>
struct TaShape {
  static constexpr int kNT = 64 * W, kWP = W / WR, kRows = 32 * WR;
  static constexpr int kChunks = HD / 8;                     // 16-byte chunks of a row
  static constexpr int kK = HD * 2 + 16;                     // bytes from row to row: an odd number of chunks
  static constexpr int kV = HD * 2 + (HD % 64 == 0 ? 64 : 0);
  static constexpr int kStage = TP * (kK + kV);
  static constexpr int kLoads = TP * kChunks / kNT;          // chunks of a thread
  static constexpr int kAcc = HD / 2;                        // accumulators of a lane
  // waves that hand their results to the first of their rows, 16 accumulators of a lane at a time
  static constexpr int kJoin = (W - WR) * 64 * kAcc * 4;
  static constexpr int kPlain = W * HD * 9 * 4;              // the plain way: 8 rows of a wave at a time
  static constexpr int kMost = kJoin > kPlain ? kJoin : kPlain;
  static constexpr int kLds = 2 * kStage > kMost ? 2 * kStage : kMost;
  static_assert(TP * kChunks % kNT == 0 && (TP == 64 || TP == 128) && TP / 32 >= kWP, "stages");
  static_assert(kK % 32 == 16 && kV % 128 == 64, "rows without bank conflicts");
};

template <typename T, int HD, int W, int WR, int TP, int NQ, int NP>
__global__ __launch_bounds__(64 * W, W / 4) void tree_kernel(PaArgs A, int wide_o) {
  typedef TaShape<HD, W, WR, TP> Sh;
  typedef typename PaType<T>::v8 v8;
  constexpr int KS = HD / 16, DB = HD / 32, WP = Sh::kWP;
  __shared__ __align__(16) uint8_t shared[Sh::kLds];
  __shared__ float ex_ml[W][32][2];
  const PagedAttnLaunch& L = A.L;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int wr = w % WR, wp = w / WR;

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
    const int row0 = rt * Sh::kRows, rows = min(Sh::kRows, sq.n * A.group - row0);
    const bool whole = t_begin == 0 && t_end == sq.tiles;
    if (t_begin == 0 && threadIdx.x == 0)
      A.share[b * A.units_per_seq + unit] =
          make_int4(blockIdx.x, whole ? (int)blockIdx.x : line_owner(at + sq.tiles - 1, total, wgs), rows, 0);
    if (rows > 0) {
      const int base = sq.len - sq.n;
      const int begin = L.window > 0 ? max(0, base - L.window + 1) : 0, end = sq.len;
      const int last_lo = L.window > 0 ? max(0, end - L.window) : 0;  // what the deepest node may see first
      const int* pages = L.table.pages + b * L.table.stride;
      const uint16_t* kp = L.kv.k + head * L.kv.head_stride;
      const uint16_t* vp = L.kv.v + head * L.kv.head_stride;
      const int s_begin = sq.start + t_begin * kTile;  // the stretch's first position
      const int stages = (t_end - t_begin) * (kTile / TP);

      // ---- the way of a stage: places (a lane has those of positions lane and lane + 64), loads, LDS
      uint32_t place[2];
      u32x4 lk[Sh::kLoads], lv[Sh::kLoads];
      uint32_t on = 0;             // of the loads in registers, those of a place
      uint64_t live[2] = {0, 0};   // of the stage in registers
      auto find = [&](int st) {
        place[0] = place[1] = kNoPlace;
        if (st < stages) {
          place[0] = pa_place(L, pages, s_begin + st * TP + lane, begin, end);
          if (TP > 64) place[1] = pa_place(L, pages, s_begin + st * TP + 64 + lane, begin, end);
        }
      };
      auto load = [&]() {
        live[0] = __ballot(place[0] != kNoPlace);
        live[1] = TP > 64 ? __ballot(place[1] != kNoPlace) : 0;
        on = 0;
        if (!(live[0] | live[1])) return;  // the pool may be empty
#pragma unroll
        for (int i = 0; i < Sh::kLoads; i++) {
          const int e = (int)threadIdx.x + Sh::kNT * i, row = e / Sh::kChunks, ch = e - row * Sh::kChunks;
          uint32_t p = __shfl((int)place[0], row & 63);
          if (TP > 64) {
            const uint32_t q = __shfl((int)place[1], row & 63);
            p = row < 64 ? p : q;
          }
          // positions without a place read the pool's first: no load is conditional
          on |= p != kNoPlace ? 1u << i : 0;
          const uint64_t o = (uint64_t)(p == kNoPlace ? 0 : p) * 8 + 8 * ch;
          lk[i] = *(const u32x4*)(kp + o);
          lv[i] = *(const u32x4*)(vp + o);
        }
      };
      find(0);
      load();
      find(1);

      // ---- queries: lane l has 8 dimensions of each 16 of row l % 32
      const int r = min(row0 + 32 * wr + c, sq.n * A.group - 1), tok = r / A.group;
      const int64_t qa = b * L.qb + tok * L.qt + (head * A.group + r - tok * A.group) * L.qh + 8 * h;
      v8 q[KS][NQ];
      float to_log2 = L.scale * kLog2e;  // what brings the row's products to log2 units
      {
        float big = 0.0f, f[KS][8];
#pragma unroll
        for (int s = 0; s < KS; s++) {
          if (NQ == 1)
            pa_load8((const T*)L.q + qa + 16 * s, A.wide_q, f[s]);  // 16 bits either way: the conversions cancel
          else if (L.dtype == kF32)
            pa_load8((const float*)L.q + qa + 16 * s, A.wide_q, f[s]);
          else if (L.dtype == kF16)
            pa_load8((const _Float16*)L.q + qa + 16 * s, A.wide_q, f[s]);
          else
            pa_load8((const __bf16*)L.q + qa + 16 * s, A.wide_q, f[s]);
#pragma unroll
          for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(f[s][i]));
        }
        float up = 1.0f;
        if (NQ > 1) {  // the largest magnitude of the row to [2^13, 2^14)
          big = fmaxf(big, __shfl_xor(big, 32));
          const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253);  // small rows: as if 2^-100
          up = __uint_as_float((uint32_t)(267 - e) << 23);
          to_log2 *= 1.0f / up;
        }
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
          for (int i = 0; i < 8; i++) f[s][i] *= up;
          pa_split<T, NQ>(f[s], q[s]);
        }
      }
      // ---- what the row sees
      const PaTree node = pa_node(pa_tree(L, b, sq.n), tok);
      const int lo = L.window > 0 ? max(0, base + node.depth - L.window + 1) : 0;

      float m = -INFINITY, l = 0.0f;
      f32x16 acc[DB];
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;

      __syncthreads();  // what the unit before left in LDS is read
      for (int st = 0; st < stages; st++) {
        uint8_t* sk = shared + (st & 1) * Sh::kStage;
        uint8_t* sv = sk + TP * Sh::kK;
        const uint64_t now[2] = {live[0], live[1]};
        if (now[0] | now[1]) {
#pragma unroll
          for (int i = 0; i < Sh::kLoads; i++) {
            const int e = (int)threadIdx.x + Sh::kNT * i, row = e / Sh::kChunks, ch = e - row * Sh::kChunks;
            const bool has = on >> i & 1;
            u32x4 x = lv[i];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = has ? x[k] : 0u;  // weights of 0 would not clear a NaN
            *(u32x4*)(sk + row * Sh::kK + 16 * ch) = lk[i];
            *(u32x4*)(sv + row * Sh::kV + 16 * ch) = x;
          }
        }
        load();  // the next stage's; its places are known
        find(st + 2);
        __syncthreads();
#pragma unroll
        for (int u0 = 0; u0 < TP / 32 / WP; u0++) {
          const int u = u0 * WP + wp, p0 = s_begin + st * TP + 32 * u;
          const uint32_t here = (uint32_t)((u < 2 ? now[0] : now[1]) >> (32 * (u & 1)));
          if (!here) continue;
          f32x16 x;
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] = 0.0f;
          const uint8_t* ka = sk + (32 * u + c) * Sh::kK + 16 * h;
#pragma unroll
          for (int s = 0; s < KS; s++) {
            const u32x4 a = *(const u32x4*)(ka + 32 * s);
#pragma unroll
            for (int k = NQ - 1; k >= 0; k--) x = TaType<T>::mfma(__builtin_bit_cast(v8, a), q[s][k], x);
          }
          float s[16];
#pragma unroll
          for (int i = 0; i < 16; i++) s[i] = x[i] * to_log2;
          if (!(here == 0xffffffffu && p0 + 31 < base && p0 >= last_lo)) {
            const uint32_t sees = tree_sees(node.above, p0, base) & tree_from(lo, p0, base) & here;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = sees >> (8 * (i >> 2) + 4 * h + (i & 3)) & 1 ? s[i] : -INFINITY;
          }
          // ---- running maximum and sum
          float top = s[0];
#pragma unroll
          for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
          top = fmaxf(top, __shfl_xor(top, 32));
          const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
          if (__any(mn > m)) {
            const float by = __builtin_amdgcn_exp2f(m - ref);
            l *= by;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
              for (int i = 0; i < 16; i++) acc[d][i] *= by;
            m = mn;
          }
          v8 pp[2][NP];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              p[i] = __builtin_amdgcn_exp2f(s[8 * k + i] - ref + PaType<T>::kOffset);
              l += p[i];
            }
            pa_split<T, NP>(p, pp[k]);
          }
          // ---- O^T += V^T P^T
          const uint8_t* va = sv + (32 * u + 4 * h + (lane >> 2 & 3)) * Sh::kV + (16 * (lane >> 4 & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const u32x2 y0 = ta_read_tr(va + 64 * d + 16 * k * Sh::kV), y1 = ta_read_tr(va + 64 * d + (16 * k + 8) * Sh::kV);
              const u32x4 a = {y0[0], y0[1], y1[0], y1[1]};
#pragma unroll
              for (int j = NP - 1; j >= 0; j--) acc[d] = TaType<T>::mfma(__builtin_bit_cast(v8, a), pp[k][j], acc[d]);
            }
        }
      }
      l += __shfl_xor(l, 32);
      float sum = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) sum += acc[d][i] * 0.0f;
      __syncthreads();  // the last stages are read
      if (__any(sum != sum)) {  // infinities and NaN among the values, or their products
        float* ex = (float*)shared + w * HD * 9;
        for (int r8 = 0; r8 < 4; r8++) {
          const int from = 32 * wr + 8 * r8;
          if (from >= rows) break;
          pa_plain<T, HD, true>(A, b, head, row0 + from, min(8, rows - from), s_begin + 32 * wp, sq.start + t_end * kTile,
                                32 * WP, sq.len, sq.n, ex, ex_ml[w], 9);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own, in order
          if (c >> 3 == r8) {
            m = ex_ml[w][c & 7][0], l = ex_ml[w][c & 7][1];
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
              for (int i = 0; i < 16; i++) acc[d][i] = ex[(32 * d + 8 * (i >> 2) + 4 * h + (i & 3)) * 9 + (c & 7)];
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
      }
      // ---- the waves of the same rows together, in order
      if constexpr (WP > 1) {
        __syncthreads();
        f32x4* ex = (f32x4*)shared;
        if (h == 0) ex_ml[w][c][0] = m, ex_ml[w][c][1] = l;
        if (wp > 0) {
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              ex[((w - WR) * DB * 4 + 4 * d + i) * 64 + lane] =
                  f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        }
        __syncthreads();
        if (wp == 0) {
          float mm = m;
#pragma unroll
          for (int k = 1; k < WP; k++) mm = fmaxf(mm, ex_ml[wr + k * WR][c][0]);
          const float ref = mm == -INFINITY ? 0.0f : mm, own = __builtin_amdgcn_exp2f(m - ref);
          l *= own;
          const bool none = !(own > 0.0f || ref != ref);  // saw nothing, or nothing of weight
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] = none ? 0.0f : acc[d][i] * own;
#pragma unroll
          for (int k = 1; k < WP; k++) {
            const int other = wr + k * WR;
            const float by = __builtin_amdgcn_exp2f(ex_ml[other][c][0] - ref);
            l += ex_ml[other][c][1] * by;
            if (by > 0.0f || ref != ref) {
#pragma unroll
              for (int d = 0; d < DB; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  const f32x4 y = ex[((other - WR) * DB * 4 + 4 * d + i) * 64 + lane];
#pragma unroll
                  for (int j = 0; j < 4; j++) acc[d][4 * i + j] += y[j] * by;
                }
            }
          }
          m = mm;
        }
      }
      const int row = 32 * wr + c;
      if (wp == 0 && row < rows) {
        if (!whole) {
          const int64_t slot = 2 * (int64_t)blockIdx.x + (t_begin == 0 ? 1 : 0);
          float* o = A.part_o + (slot * A.slots + row) * HD + 4 * h;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              *(f32x4*)(o + 32 * d + 8 * i) = f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
          if (h == 0) A.part_ml[slot * A.slots + row] = make_float2(m, l);
        } else {
          const int hh = head * A.group + r - tok * A.group;
          const int64_t o = b * L.ob + tok * L.ot + hh * L.oh + 4 * h;
          const bool none = m == -INFINITY && l == 0.0f;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              float y[4];
#pragma unroll
              for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : acc[d][4 * i + j] / l;
              pa_store4(L.out, L.dtype, o + 32 * d + 8 * i, wide_o, y);
            }
          if (L.lse && h == 0)
            L.lse[((int64_t)b * L.n_new + tok) * L.heads + hh] =
                none ? -INFINITY : (m - PaType<T>::kOffset + log2f(l)) * 0.69314718055994531f;
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

template <typename T, int HD, int W, int WR, int TP, int NQ, int NP>
hipError_t ta_launch(const PagedAttnLaunch& L) {
  PaArgs A = pa_args(L, 32 * WR);
  const int64_t units = (int64_t)A.units_per_seq * L.table.seqs;
  const int64_t tiles = ((int64_t)L.table.width * L.kv.page_size + kTile - 1) / kTile;
  const int64_t most = units * (tiles > 0 ? tiles : 1);
  A.wgs = (int)(most < kTaWgs ? most : kTaWgs);
  pa_workspace(A, HD);
  const int v = L.dtype == kF32 ? 4 : 2;  // four values are stored together
  const int wide_o = ((uintptr_t)L.out & (v == 4 ? 15 : 7)) == 0 && L.ob % 4 == 0 && L.ot % 4 == 0 && L.oh % 4 == 0;
  hipLaunchKernelGGL((tree_kernel<T, HD, W, WR, TP, NQ, NP>), dim3(A.wgs), dim3(64 * W), 0, L.stream, A, wide_o);
  if (tiles > 1)
    hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3((unsigned)units, A.slots), dim3(256), 0, L.stream, A);
  return hipGetLastError();
}

// Units of as many rows as there are, up to what a workgroup's registers hold: 32 a wave, of eight waves on two a SIMD, or
// where a row takes more registers (heads of 256, queries in three pieces) of four.
template <typename T, int HD, int NQ, int NP>
hipError_t ta_launch_rows(const PagedAttnLaunch& L) {
  const int rows = L.n_new * (L.heads / L.kv.n_kv);
  if constexpr (HD > 128 || NQ > 2) {
    if (rows > 64) return ta_launch<T, HD, 4, 4, 64, NQ, NP>(L);
    return ta_launch<T, HD, 4, 2, 64, NQ, NP>(L);
  } else {
    constexpr int kTP = (HD == 128 && NQ == 2) ? 64 : 128;  // registers for a stage of 64 beside the queries' pieces
    if (rows > 128) return ta_launch<T, HD, 8, 8, kTP, NQ, NP>(L);
    if (rows > 64) return ta_launch<T, HD, 8, 4, kTP, NQ, NP>(L);
    return ta_launch<T, HD, 8, 2, 128, NQ, NP>(L);
  }
}

template <typename T, int HD>
hipError_t ta_launch_hd(const PagedAttnLaunch& L) {
  constexpr int kMany = PaType<T>::kPieces;
  if ((size_t)L.n_new * (L.heads / L.kv.n_kv) <= ta_few(HD)) return pa_launch_hd<T, HD, true>(L);
  // a weight's pieces: two are within 2^-17 of it (bf16), far below a rounding of a 16-bit output
  if (L.dtype == PaType<T>::kId) return ta_launch_rows<T, HD, 1, 2>(L);
  return ta_launch_rows<T, HD, kMany, kMany>(L);
}

template <typename T>
hipError_t ta_launch_type(const PagedAttnLaunch& L) {
  switch (L.kv.hd) {
    case 32: return ta_launch_hd<T, 32>(L);
    case 64: return ta_launch_hd<T, 64>(L);
    case 96: return ta_launch_hd<T, 96>(L);
    case 128: return ta_launch_hd<T, 128>(L);
    default: return ta_launch_hd<T, 256>(L);
  }
}

}  // namespace
}  // namespace nrq
