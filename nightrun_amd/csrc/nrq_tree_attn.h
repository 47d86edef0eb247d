// Attention of a tree's nodes over a paged cache (include/nrq_tree.h, nrq_dev_tree_attention): the kernels, instantiated
// per cache type in nrq_tree_f16.hip and nrq_tree_bf16.hip. What they have in common with the attention of a sequence's last tokens (the line
// of tiles and its stretches, pieces of f32 values, the plain way for infinities) is in nrq_paged.h.
//
// With R rows (nodes x query heads of a KV head) a position of a KV head costs 4 R head_dim operations for 4 head_dim bytes,
// R operations a byte: groups of 32 rows that each read the keys and values for themselves ask the L2 for
// more than it delivers (24 sequences of 64 nodes, f16: 824 us so, 174 here). So a unit is up to 256 rows, and its keys and values
// pass through LDS once for all of them: stage by stage, the next one on its way from memory to LDS while one is multiplied.
//
// A wave owns 32 rows; where there are fewer of those than waves, each takes a part of each stage's positions, and their results
// are added up in LDS at the end of a stretch. Per 32 positions:
//   S^T = K Q^T on 32x32x16 matrix instructions, queries in registers: lane l gets row l % 32 at positions
//   8 i + 4 (l / 32) + j, which is the order in which P^T goes into the second product,
//   O^T += V^T P^T, with V^T read transposed from LDS (four positions of one dimension a lane).
// Chunks of a stage's rows are dealt round the banks (key_chunk, value_chunk), so that neither read meets a bank twice: the counters
// show no conflicts.
//
// What bounds it. Two sequences of 65,536 and 131,072 positions by 64 nodes (256 rows a KV head of 128, f16; 805 MB, 206 GFLOP, 309 with the
// weights in two pieces) take 351 to 358 us, 10 of them the join: the matrix units work half of the clocks, vector instructions the other half, and the
// clock is down to 1.75 GHz, the power limit; without its loads it would take 300. Orders of instructions, priorities and stages that
// keep both busier change nothing there. 64 rows a wave halve the reads of LDS but leave the 256 registers that
// vector instructions reach: 415. 24 sequences of up to 6000 by 32 nodes (128 rows, bf16, 307 MB) 112 to 118 us, 15 of them the join: the
// matrix units work 40% of the clocks, vector instructions 45%; with the weights in two pieces instead of three, which left them 16 bits, 99. In f16
// 105. What else it takes is units' beginnings and ends, one after the other: length, pages, queries and first stage, and parts that are
// written and read again. 13 sequences under a window of 4096 by 25 nodes, f32 queries in two pieces (178 MB) 72 to 77: the same, and two to six
// registers that spill (f32 queries over an f16 cache, heads of 128: the pieces of both leave no room). One sequence of 1001 positions by 8
// nodes 13.7: two launches, one tile a workgroup, half of whose waves have no rows.
#pragma once

#include "nrq_paged.h"
#include "nrq_tree_launch.h"

namespace nrq {

constexpr int kTaCus = 256;
// What the beginning and the end of a unit cost, in tiles: stretches of many short units are as long as those of a few long ones. 24
// sequences of 250 to 6000 positions by 64 nodes take 214, 182, 174, 174 us with 0, 1, 2, 3, 181 with 5 (f16), by 32 nodes 122, 107, 105, 105,
// 108 and 128, 116, 117, 118, 121 (bf16); 13 of one length 105, 104, 102, 102, 104.
constexpr int kTaSetup = 3;
// Workgroups of a unit, on average, from which on the join takes a row a workgroup, 16 stretches side by side, else four rows, four
// stretches side by side: one KV head over 131,072 positions by 4 nodes 38 us so, 56 the other way (93 with one after the
// other); two sequences of 8 heads (16 workgroups a unit) 358 and 354, 24 by 32 nodes (three) 128 and 105.
constexpr int kTaShared = 32;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct TaType;
template <>
struct TaType<_Float16> {
  static constexpr float kRoom = 3.0f;  // weights up to 2^15
  typedef PaType<_Float16>::v8 v8;
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct TaType<__bf16> {
  static constexpr float kRoom = 16.0f;  // as many bits at any size
  typedef PaType<__bf16>::v8 v8;
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Four positions of one dimension: of 16 lanes, lanes 4 r .. 4 r + 3 name 16 consecutive values of row r, lane i gets
// the i-th of each of the four rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 ta_read_tr(uint32_t at) {
  typedef __attribute__((address_space(3))) s16x4* lds;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)at));
}
__device__ __forceinline__ u32x4 ta_read(uint32_t at) { return *(__attribute__((address_space(3))) u32x4*)at; }

__device__ const uint32_t ta_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// 16 bytes a lane from memory to LDS, lane after lane from byte address m0 (wave-uniform)
__device__ __forceinline__ void ta_dma16(const void* g, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0), "v"(g) : "memory");
}

// The pieces of eight weights, as pa_split() has them, in fewer instructions: conversions by twos, the rest of a
// value in one fused step.
template <typename T, int N>
__device__ __forceinline__ void ta_split(const float* f, typename PaType<T>::v8* out) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = f[i];
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const t2 x = __builtin_convertvector((f2{r[i], r[i + 1]}), t2);
      out[k][i] = x[0], out[k][i + 1] = x[1];
      if (k + 1 < N) r[i] = fmaf((float)x[0], -1.0f, r[i]), r[i + 1] = fmaf((float)x[1], -1.0f, r[i + 1]);
    }
}

// W waves, WR of them side by side over the rows, TP positions of a stage.
template <int HD, int W, int WR, int TP>
struct TaShape {
  static constexpr int kNT = 64 * W, kWP = W / WR, kRows = 32 * WR;
  static constexpr int kChunks = HD / 8;                     // 16-byte chunks of a row
  static constexpr int kRow = HD * 2;                        // bytes
  static constexpr int kStage = 2 * TP * kRow;               // keys, then values
  static constexpr int kLoads = TP * kChunks / kNT;          // chunks of a thread, of keys and of values
  static constexpr int kAcc = HD / 2;                        // accumulators of a lane
  // waves that hand their results to the first of their rows
  static constexpr int kJoin = (W - WR) * 64 * kAcc * 4;
  static constexpr int kPlain = W * HD * 9 * 4;              // the plain way: 8 rows of a wave at a time
  static constexpr int kMost = kJoin > kPlain ? kJoin : kPlain;
  static constexpr int kLds = 2 * kStage > kMost ? 2 * kStage : kMost;
  static_assert(TP * kChunks % kNT == 0 && (TP == 64 || TP == 128) && TP / 32 >= kWP, "stages");

  // Where chunk c of a row's keys lies in the row: 16 rows from any on have it on 16 different places of the 64 banks.
  static __device__ __forceinline__ int key_chunk(int row, int c) {
    if constexpr (HD % 128 == 0) return c ^ (row & 15);
    if constexpr (HD == 64) return c ^ (row >> 1 & 7);
    if constexpr (HD == 32) return c ^ (row >> 2 & 3);
    const int x = c + (row >> 2 & 3);  // rows of 12 chunks
    return x < kChunks ? x : x - kChunks;
  }
  // The chunk of a row's keys that lies at place p.
  static __device__ __forceinline__ int key_at(int row, int p) {
    if constexpr (HD != 96) return key_chunk(row, p);
    const int x = p - (row >> 2 & 3);
    return x < 0 ? x + kChunks : x;
  }
  // The same for values, both ways: the 64 bytes that hold a dimension of four rows from a multiple of 4 on lie in
  // four different quarters of the banks.
  static __device__ __forceinline__ int value_chunk(int row, int c) {
    if constexpr (HD % 128 == 0) return c ^ (row & 3) << 2;
    if constexpr (HD == 64) return c ^ (row >> 1 & 1) << 2;
    return c;
  }
};

// Waves of a SIMD: registers for the accumulators and the queries' pieces.
constexpr int ta_waves(int hd, int nq) { return hd > 128 || nq > 2 ? 1 : 2; }

template <typename T, int HD, int W, int WR, int TP, int NQ>
__global__ __launch_bounds__(64 * W, ta_waves(HD, NQ)) void tree_kernel(PaArgs A, int wide_o) {
  typedef TaShape<HD, W, WR, TP> Sh;
  typedef typename PaType<T>::v8 v8;
  constexpr int NP = PaType<T>::kPieces;  // of a weight: f32 values, as in nrq_paged.h
  constexpr int KS = HD / 16, DB = HD / 32, WP = Sh::kWP;
  __shared__ __align__(512) uint8_t shared[Sh::kLds];  // rows of a stage begin at multiples of their size
  __shared__ float ex_ml[W][32][2];
  const PagedAttnLaunch& L = A.L;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int wr = w % WR, wp = w / WR;

  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)shared;

  const PaLine line = pa_line(A, blockIdx.x);
  const int total = line.total, wgs = line.wgs;
  if ((int)blockIdx.x >= wgs) return;
  int at = line.at, first = line.first, b = line.b;
  const int stop = line_start(blockIdx.x + 1, total, wgs);
  while (at < stop) {
    const SeqSpan sq = pa_seq(L, b);
    // a unit's place in the line: what its beginning costs, then its tiles
    const int length = sq.tiles + A.setup, unit = (at - first) / length;
    const int v_begin = at - first - unit * length, v_end = min(length, v_begin + (stop - at));
    const int t_begin = max(0, v_begin - A.setup), t_end = max(0, v_end - A.setup);
    const int head = unit / A.row_tiles, rt = unit - head * A.row_tiles;
    const int row0 = rt * Sh::kRows, rows = min(Sh::kRows, sq.n * A.group - row0);
    const bool whole = t_begin == 0 && t_end == sq.tiles;
    if (t_begin == 0 && t_end > 0 && threadIdx.x == 0)
      A.share[b * A.units_per_seq + unit] =
          make_int4(blockIdx.x, whole ? (int)blockIdx.x : line_owner(first + (unit + 1) * length - 1, total, wgs), rows, 0);
    if (rows > 0 && t_begin < t_end) {
      const int base = sq.len - sq.n;
      const int begin = L.window > 0 ? max(0, base - L.window + 1) : 0, end = sq.len;
      const int last_lo = L.window > 0 ? max(0, end - L.window) : 0;  // what the deepest node may see first
      const int* pages = L.table.pages + b * L.table.stride;
      const uint16_t* kp = L.kv.k + head * L.kv.head_stride;
      const uint16_t* vp = L.kv.v + head * L.kv.head_stride;
      const int s_begin = sq.start + t_begin * kTile;  // the stretch's first position
      const int stages = (t_end - t_begin) * (kTile / TP);

      // ---- the way of a stage: a lane asks for the pages of positions lane and lane + 64, one stage later has their
      // places and the loads go out, another stage later what they brought goes to LDS. The pages are asked for before
      // the loads and looked at behind them: loads come back in order, and a wait for a page right after it is asked for were one for
      // all loads before it.
      constexpr int kHalf = TP / 64;
      uint32_t column[kHalf], within[kHalf], page[kHalf], place[kHalf];
      uint64_t asked[kHalf];
      const uint32_t size = L.kv.page_size, steps = TP / size, rest = TP - steps * size;
#pragma unroll
      for (int i = 0; i < kHalf; i++) {
        const uint32_t t = s_begin + 64 * i + lane;
        column[i] = t / size, within[i] = t - column[i] * size;
      }
      uint64_t live[2] = {0, 0};   // of the stage on its way
      auto ask = [&](int st) {
#pragma unroll
        for (int i = 0; i < kHalf; i++) {
          const int t = s_begin + st * TP + 64 * i + lane;
          const bool ok = st < stages && t >= begin && t < end && column[i] < (uint32_t)L.table.width;
          asked[i] = __ballot(ok);
          page[i] = 0;
          if (asked[i]) page[i] = pages[ok ? column[i] : 0];  // where any is, the table has a column
        }
      };
      auto look = [&]() {  // behind ask()
#pragma unroll
        for (int i = 0; i < kHalf; i++) {
          const bool ok = (asked[i] >> lane & 1) && page[i] < (uint32_t)L.kv.n_pages;
          place[i] = ok ? page[i] * L.kv.page_stride8 + within[i] * L.kv.pos_stride8 : kNoPlace;
          column[i] += steps, within[i] += rest;
          if (within[i] >= size) within[i] -= size, column[i]++;
        }
      };
      auto load = [&](int st) {
        live[0] = __ballot(place[0] != kNoPlace);
        live[1] = kHalf > 1 ? __ballot(place[kHalf - 1] != kNoPlace) : 0;
        if (!(live[0] | live[1])) return;
        const uint32_t to = lds + (st & 1) * Sh::kStage + w * 1024;
#pragma unroll
        for (int i = 0; i < Sh::kLoads; i++) {
          const int e = (int)threadIdx.x + Sh::kNT * i, row = e / Sh::kChunks, at_ = e - row * Sh::kChunks;
          uint32_t p = __shfl((int)place[0], row & 63);
          if (kHalf > 1) {
            const uint32_t p1 = __shfl((int)place[kHalf - 1], row & 63);
            p = row < 64 ? p : p1;
          }
          // positions without a place are zeros: weights of 0 would not clear what a page holds, a NaN
          const uint64_t o = (uint64_t)p * 8;
          const uint16_t* fk = p == kNoPlace ? (const uint16_t*)ta_zeros : kp + (o + 8 * Sh::key_at(row, at_));
          const uint16_t* fv = p == kNoPlace ? (const uint16_t*)ta_zeros : vp + (o + 8 * Sh::value_chunk(row, at_));
          ta_dma16(fk, to + Sh::kNT * 16 * i);
          ta_dma16(fv, to + Sh::kNT * 16 * i + TP * Sh::kRow);
        }
      };
      __syncthreads();  // what the unit before left in LDS is read
      ask(0);
      // ---- queries: lane l has 8 dimensions of each 16 of row l % 32
      const int r = min(row0 + 32 * wr + c, sq.n * A.group - 1), tok = r / A.group;
      const int64_t qa = b * L.qb + tok * L.qt + (head * A.group + r - tok * A.group) * L.qh + 8 * h;
      v8 q[KS][NQ];
      PaTree node;  // what the row sees
      float to_log2 = fabsf(L.scale) * kLog2e;  // what brings the row's products to log2 units; its sign goes into the queries
      {
        float big = 0.0f, f[KS][8];
        const int parent = pa_parent(L, b, sq.n);
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
        }
        // pages, parents and queries are on their way together; the first stage's loads go out as soon as its pages are there
        __builtin_amdgcn_sched_barrier(0);
        look();
        ask(1);
        load(0);
        __builtin_amdgcn_sched_barrier(0);
        node = pa_node(pa_tree(L, parent, sq.n), tok);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(f[s][i]));
        float up = L.scale < 0.0f ? -1.0f : 1.0f;
        if (NQ > 1) {  // the largest magnitude of the row to [2^13, 2^14)
          big = fmaxf(big, __shfl_xor(big, 32));
          const int e = min(max((int)(__float_as_uint(big) >> 23), 27), 253);  // small rows: as if 2^-100
          const float by = __uint_as_float((uint32_t)(267 - e) << 23);
          up *= by;
          to_log2 *= 1.0f / by;
        }
        if (to_log2 == 0.0f) up = 0.0f, to_log2 = 1.0f;  // times 0, a masked score were NaN
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
          for (int i = 0; i < 8; i++) f[s][i] *= up;
          pa_split<T, NQ>(f[s], q[s]);
        }
        // they are here before the stages begin: a wait for them in the loop would be one for the next stage's loads too
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int k = 0; k < NQ; k++) asm volatile("" : "+v"(q[s][k]));
      }
      const int lo = L.window > 0 ? max(0, base + node.depth - L.window + 1) : 0;

      float m = -INFINITY, l = 0.0f;
      f32x16 acc[DB];
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;

      for (int st = 0; st < stages; st++) {
        const uint32_t sk = lds + (st & 1) * Sh::kStage, sv = sk + TP * Sh::kRow;
        const uint64_t now[2] = {live[0], live[1]};
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of the stage is there
        __syncthreads();                                  // and so are the others', who have read the stage before it
        look();
        ask(st + 2);
        load(st + 1);
        if (!(now[0] | now[1]) || 32 * wr >= rows) continue;
        constexpr int US = TP / 32 / WP;  // of 32 positions, the wave's
        // the first half of the keys is read ahead, the second while the first is multiplied
        constexpr int KH = KS / 2;
        u32x4 ka[KH], kb[KH];
        auto read_k = [&](int u, int half, u32x4* k) {
          const int row = 32 * u + c;
          const uint32_t line = sk + row * Sh::kRow;
#pragma unroll
          for (int s = 0; s < KH; s++) {
            const int ch = 2 * (KH * half + s);
            if constexpr (HD == 96)
              k[s] = ta_read(line + 16 * Sh::key_chunk(row, ch + h));
            else  // the chunk's bits and the row's
              k[s] = ta_read((line + 16 * Sh::key_chunk(row, h)) ^ (16 * ch));
          }
        };
        read_k(wp, 0, ka);
#pragma unroll 1
        for (int u0 = 0; u0 < US; u0++) {
          const int u = u0 * WP + wp, p0 = s_begin + st * TP + 32 * u;
          const uint32_t here = (uint32_t)((u < 2 ? now[0] : now[1]) >> (32 * (u & 1)));
          f32x16 x;
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] = 0.0f;
          read_k(u, 1, kb);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int k = NQ - 1; k >= 0; k--)
              x = TaType<T>::mfma(__builtin_bit_cast(v8, s < KH ? ka[s % KH] : kb[s % KH]), q[s][k], x);
          // reads run ahead of the products that take them: the first values' over the softmax, the next keys' over the values'
          const int vrow = 4 * h + (lane >> 2 & 3);  // its low bits are the same 8 rows on
          const uint32_t va = sv + (32 * u + vrow) * Sh::kRow + (lane & 1) * 8 +
                              16 * Sh::value_chunk(vrow, (lane >> 4 & 1) * 2 + (lane >> 1 & 1));
          u32x4 vt[2][2];
          auto read_v = [&](int d) {
            const uint32_t y = HD == 96 ? va + 64 * d : va ^ (64 * d);
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const u32x2 y0 = ta_read_tr(y + 16 * k * Sh::kRow), y1 = ta_read_tr(y + (16 * k + 8) * Sh::kRow);
              vt[d & 1][k] = u32x4{y0[0], y0[1], y1[0], y1[1]};
            }
          };
          read_v(0);
          __builtin_amdgcn_sched_barrier(0);
          if (!(here == 0xffffffffu && p0 + 31 < base && p0 >= last_lo)) {
            const uint32_t sees = tree_sees(node.above, p0, base) & tree_from(lo, p0, base) & here, mine = sees >> (4 * h);
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = mine & 1u << (8 * (i >> 2) + (i & 3)) ? x[i] : -INFINITY;
          }
          // ---- running maximum and sum
          float top = x[0];
#pragma unroll
          for (int i = 1; i < 16; i++) top = fmaxf(top, x[i]);
          top = fmaxf(top, __shfl_xor(top, 32));
          // the weights' unit 2^m follows the maximum only where it is left behind by more than the weights' type has room for:
          // the accumulators are brought to another unit a few times a stretch, not in every other tile
          const float mn = fmaxf(m, top * to_log2);
          const bool behind = __any(mn > m + TaType<T>::kRoom);
          const float ref = behind ? (mn == -INFINITY ? 0.0f : mn) : (m == -INFINITY ? 0.0f : m);
          if (behind) {
            const float by = __builtin_amdgcn_exp2f(m - ref);
            l *= by;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
              for (int i = 0; i < 16; i++) acc[d][i] *= by;
            m = mn;
          }
          const float less = PaType<T>::kOffset - ref;
          v8 pp[2][NP];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              p[i] = __builtin_amdgcn_exp2f(fmaf(x[8 * k + i], to_log2, less));
              l += p[i];
            }
            ta_split<T, NP>(p, pp[k]);
          }
          // ---- O^T += V^T P^T
          if (u0 + 1 < US) read_k(u + WP, 0, ka);
#pragma unroll
          for (int d = 0; d < DB; d++) {
            if (d + 1 < DB) read_v(d + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
              for (int j = NP - 1; j >= 0; j--) acc[d] = TaType<T>::mfma(__builtin_bit_cast(v8, vt[d & 1][k]), pp[k][j], acc[d]);
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
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] = pa_less(acc[d][i], own);
#pragma unroll
          for (int k = 1; k < WP; k++) {
            const int other = wr + k * WR;
            const float by = __builtin_amdgcn_exp2f(ex_ml[other][c][0] - ref);
            l += ex_ml[other][c][1] * by;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const f32x4 y = ex[((other - WR) * DB * 4 + 4 * d + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[d][4 * i + j] += pa_less(y[j], by);
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
          const float by = 1.0f / l;
#pragma unroll
          for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              float y[4];
#pragma unroll
              for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : acc[d][4 * i + j] * by;
              pa_store4(L.out, L.dtype, o + 32 * d + 8 * i, wide_o, y);
            }
          if (L.lse && h == 0)
            L.lse[((int64_t)b * L.n_new + tok) * L.heads + hh] =
                none ? -INFINITY : (m - PaType<T>::kOffset + log2f(l)) * 0.69314718055994531f;
        }
      }
    }
    at += v_end - v_begin;
    if (at == first + length * A.units_per_seq) {
      first = at;
      b++;
    }
  }
}

// The stretches of a unit that several workgroups shared: 16 lanes a row and G groups of them, each of which takes every
// G-th stretch; what they have is added up in order.
template <typename T, int HD, int G>
__global__ __launch_bounds__(256) void tree_join_kernel(PaArgs A, int wide_o) {
  constexpr int E = HD / 16, F = E % 4 ? 2 : 4;  // dimensions of a lane, F side by side
  constexpr int R = 16 / G;                      // rows
  __shared__ float ex_o[G > 1 ? G : 1][R][G > 1 ? HD : 1], ex_l[G][R];
  const PagedAttnLaunch& L = A.L;
  const int u = blockIdx.x, b = u / A.units_per_seq, unit = u - b * A.units_per_seq;
  const int4 share = A.share[u];
  const int c = threadIdx.x & 15, g = (threadIdx.x >> 4) % G, rw = threadIdx.x / (16 * G), r = R * blockIdx.y + rw;
  const int w0 = share.x, n = share.y - w0 + 1;
  if (n < 2 || R * (int)blockIdx.y >= share.z) return;
  const bool on = r < share.z;
  const int head = unit / A.row_tiles, rr = (unit - head * A.row_tiles) * A.per + r;
  auto slot = [&](int k) { return (int64_t)(2 * (w0 + k) + (k == 0 ? 1 : 0)) * A.slots + (on ? r : 0); };
  float mm = -INFINITY;
  for (int k = c; k < n; k += 16) mm = fmaxf(mm, A.part_ml[slot(k)].x);
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) mm = fmaxf(mm, __shfl_xor(mm, x, 16));
  const float ref = mm == -INFINITY ? 0.0f : mm;
  float o[E], l = 0;
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = 0;
#pragma unroll 4
  for (int k = g; k < n; k += G) {
    const int64_t s = slot(k);
    const float2 x = A.part_ml[s];
    const float by = __builtin_amdgcn_exp2f(x.x - ref);
    l += x.y * by;
    const float* p = A.part_o + s * HD + F * c;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] += pa_less(p[e / F * 16 * F + e % F], by);
  }
  if constexpr (G > 1) {
#pragma unroll
    for (int e = 0; e < E; e++) ex_o[g][rw][16 * e + c] = o[e];
    if (c == 0) ex_l[g][rw] = l;
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int k = 1; k < G; k++) {
      l += ex_l[k][rw];
#pragma unroll
      for (int e = 0; e < E; e++) o[e] += ex_o[k][rw][16 * e + c];
    }
  }
  if (!on) return;
  const int tok = rr / A.group, h = head * A.group + rr - tok * A.group;
  const bool none = mm == -INFINITY && l == 0.0f;
  const float by = 1.0f / l;
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = none ? 0.0f : o[e] * by;
  const int64_t at = b * L.ob + tok * L.ot + h * L.oh + F * c;
#pragma unroll
  for (int e = 0; e < E; e += F) {
    if constexpr (F == 4) {
      pa_store4(L.out, L.dtype, at + e / F * 16 * F, wide_o, o + e);
    } else {
#pragma unroll
      for (int i = 0; i < F; i++) pa_store(L.out, L.dtype, at + e / F * 16 * F + i, o[e + i]);
    }
  }
  if (L.lse && c == 0)
    L.lse[((int64_t)b * L.n_new + tok) * L.heads + h] =
        none ? -INFINITY : (mm - PaType<T>::kOffset + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int HD, int W, int WR, int TP, int NQ>
hipError_t ta_launch(const PagedAttnLaunch& L) {
  PaArgs A = pa_args(L, 32 * WR);
  const int64_t units = (int64_t)A.units_per_seq * L.table.seqs;
  const int64_t tiles = ((int64_t)L.table.width * L.kv.page_size + kTile - 1) / kTile;
  A.setup = kTaSetup;
  const int64_t most = units * ((tiles > 0 ? tiles : 1) + A.setup);
  constexpr int kWgs = kTaCus * ta_waves(HD, NQ) * 4 / W;  // what the card holds
  A.wgs = (int)(most < kWgs ? most : kWgs);
  pa_workspace(A, HD);
  const int v = L.dtype == kF32 ? 4 : 2;  // four values are stored together
  const int wide_o = ((uintptr_t)L.out & (v == 4 ? 15 : 7)) == 0 && L.ob % 4 == 0 && L.ot % 4 == 0 && L.oh % 4 == 0;
  hipLaunchKernelGGL((tree_kernel<T, HD, W, WR, TP, NQ>), dim3(A.wgs), dim3(64 * W), 0, L.stream, A, wide_o);
  if (tiles > 1 && A.wgs >= kTaShared * units)
    hipLaunchKernelGGL((tree_join_kernel<T, HD, 16>), dim3((unsigned)units, A.slots), dim3(256), 0, L.stream, A, wide_o);
  else if (tiles > 1)
    hipLaunchKernelGGL((tree_join_kernel<T, HD, 4>), dim3((unsigned)units, (A.slots + 3) / 4), dim3(256), 0, L.stream, A, wide_o);
  return hipGetLastError();
}

// Units of as many rows as there are, up to what a workgroup's registers hold: 32 a wave, of eight waves on two a SIMD, or
// where a row takes more registers (heads of 256, queries in three pieces) of four.
template <typename T, int HD, int NQ>
hipError_t ta_launch_rows(const PagedAttnLaunch& L) {
  const int rows = L.n_new * (L.heads / L.kv.n_kv);
  // Units of as many rows as leave each workgroup three tiles, as far as the table goes (the lengths are on the device). One sequence by 64
  // nodes of 4 heads: 4000 positions 35 us in units of 256 rows, 28 of 64; 16,000 48 and 50; 32 nodes, 8000 positions 35 in units of
  // 128 and 29 of 64. So a table far wider than its sequences are long costs short ones: those 4000 positions take 37 in one for 131,072.
  const int64_t tiles = (int64_t)L.table.seqs * L.kv.n_kv * (((int64_t)L.table.width * L.kv.page_size + kTile - 1) / kTile);
  auto fills = [&](int per, int wgs) { return tiles * ((rows + per - 1) / per) >= 3 * wgs; };
  if constexpr (HD > 128 || NQ > 2) {
    if (rows > 64 && fills(128, kTaCus)) return ta_launch<T, HD, 4, 4, 64, NQ>(L);
    return ta_launch<T, HD, 4, 2, 64, NQ>(L);
  } else {
    // More than 128 rows: one workgroup of eight waves a CU (two long sequences by 64 nodes 359 us, in two units of 128 rows 414, in four
    // of 64 531). Else two of four waves, one of which multiplies while the other begins or ends a unit (24 sequences by 32 nodes
    // in f16 105 us, with one of eight waves 106.5; in bf16 118 and 116).
    constexpr int kTP = HD == 128 || HD == 96 ? 64 : 128;
    if (rows > 128 && fills(256, kTaCus)) return ta_launch<T, HD, 8, 8, HD == 96 ? 128 : kTP, NQ>(L);
    if (rows > 64 && fills(128, 2 * kTaCus)) return ta_launch<T, HD, 4, 4, kTP, NQ>(L);
    return ta_launch<T, HD, 4, 2, kTP, NQ>(L);
  }
}

template <typename T, int HD>
hipError_t ta_launch_hd(const PagedAttnLaunch& L) {
  if (L.dtype == PaType<T>::kId) return ta_launch_rows<T, HD, 1>(L);
  return ta_launch_rows<T, HD, PaType<T>::kPieces>(L);
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
