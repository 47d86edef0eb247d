// The MXFP4 product over many tokens: tiles of 128 rows of w by 128 tokens.
//
// y[b][r] = sum over blocks k of 2^(es + et - 254) * sum over the block's 32 columns of the E2M1
// products, summed in 32 bits by the scaled matrix instruction (16 x 16 x 128, a scale byte per row and
// block); rounded once, at the store. 2048 f32 tokens by 16384 x 2048, their quantization included, take
// 61 us: 2.2 PFLOP/s and 2.2 TB/s of f32 outputs; 4096 x 4096 by 4096 tokens takes 75 us, 1.8 PFLOP/s. The
// matrix units are busy a third of that: a step's loads, its reads from LDS (32 KiB for 128 x 128 x
// 128) and its products overlap only as far as the CU's two workgroups drift apart.
//
// Up to 384 columns one kernel takes a tile a workgroup, in steps of 256 columns; beyond,
// the persistent one below. In the first a stage holds 256 columns (128 bytes) of the tile's 128 + 128 rows, 32 KiB; two
// stages take turns, filled by direct loads to LDS while the other is
// multiplied, two workgroups a CU. 16-byte chunk c of row r lies at c ^ (r / 2 & 7): the 16
// rows that a matrix instruction's quarter reads at one chunk fall on 16 different
// places of the 64 banks. A wave multiplies 64 rows by 64 tokens; of lane l's
// two steps in a stage, step s takes block 2 (l / 16) + s, so that both scale bytes of a
// row come as one 16-bit load and the instruction picks the byte. Chunks behind
// the last column come from zeros; rows behind the last are the last once more and are not stored.
#include "nrq_serve_launch.h"

#include <type_traits>

namespace nrq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kGemmTile = 128;

__device__ const uint32_t mx_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// 16 bytes a lane from memory to LDS, lane after lane from byte address m0 (wave-uniform)
__device__ __forceinline__ void mx_dma16(const void* g, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0), "v"(g) : "memory");
}

template <int S>
__device__ __forceinline__ f32x4 mx_step(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  const i32x8 x = {a.x, a.y, a.z, a.w, 0, 0, 0, 0}, y = {b.x, b.y, b.z, b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, S, sa, S, sb);
}

// Four outputs past the caches, which w and the tokens fill: 16384 x 2048 at 2048 tokens takes 92
// us so, 117 through them.
template <typename T>
__device__ __forceinline__ void mx_put(void* y, int64_t at, f32x4 v) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  const t4 o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  __builtin_nontemporal_store(o, (t4*)((T*)y + at));
}

template <typename T>
__device__ __forceinline__ void mx_out(void* y, int64_t at, int n, bool wide, f32x4 v) {
  if (wide && n >= 4) {
    mx_put<T>(y, at, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) ((T*)y)[at + i] = (T)v[i];
  }
}

// Workgroups go round the eight XCDs; each XCD gets a run of the tiles, of which its workgroups
// take every step-th. Tiles go by groups of up to 16 row tiles, within a group by tokens, and for the
// same tokens by rows: so an XCD keeps its rows of w in its L2, and what it writes at a
// time lies together (by tokens first, 16384 x 2048 at 2048 tokens takes 94 us, so 75).
struct GemmRun {
  int first, stop, step;
};
__device__ __forceinline__ GemmRun gemm_run(int all) {  // the grid is a multiple of 8
  const int x = blockIdx.x & 7, start = x * (all >> 3) + min(x, all & 7);
  return GemmRun{start + (int)(blockIdx.x >> 3), start + (all >> 3) + (x < (all & 7) ? 1 : 0), (int)(gridDim.x >> 3)};
}
struct GemmTile {
  int r, b;
};
__device__ __forceinline__ GemmTile gemm_tile(int t, int row_tiles, int tok_tiles) {
  const int group = min(16, (row_tiles + 7) >> 3), q = t / (group * tok_tiles), i = t - q * group * tok_tiles;
  const int rows = min(group, row_tiles - q * group), b = i / rows;
  return GemmTile{q * group + i - b * rows, b};
}

template <typename T>
__global__ __launch_bounds__(256, 2) void mx_gemm_kernel(MxMatmul L, int row_tiles, int tok_tiles, int wide) {
  __shared__ __align__(16) uint8_t stage[2][256][128];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, tiles_k = (blocks + 7) / 8;
  const GemmRun run = gemm_run(row_tiles * tok_tiles);
  if (run.first >= run.stop) return;
  const GemmTile tile = gemm_tile(run.first, row_tiles, tok_tiles);
  const int r0 = tile.r * kGemmTile, b0 = tile.b * kGemmTile;

  // this lane's chunks of a stage: row 32 j + 8 w + lane / 8, j < 4 of w, then of the tokens
  const int sub = 8 * w + (lane >> 3), chunk = (lane & 7) ^ (((w & 1) << 2 | lane >> 4) & 7);
  const uint8_t* src[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int r = 32 * (j & 3) + sub;
    src[j] = j < 4 ? L.w + (int64_t)min(r0 + r, L.rows - 1) * blocks * 16 : L.x + (int64_t)min(b0 + r, L.batch - 1) * blocks * 16;
    src[j] += chunk * 16;
  }
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&stage[0][0][0] + (uint32_t)w * 1024u);
  auto fill = [&](int kt) {
    const bool live = 8 * kt + chunk < blocks;
    const uint32_t to = base + (uint32_t)(kt & 1) * 32768u;
#pragma unroll
    for (int j = 0; j < 8; j++) mx_dma16(live ? src[j] + (int64_t)kt * 128 : (const uint8_t*)mx_zeros, to + (uint32_t)j * 4096u);
  };
  // scale bytes of this wave's rows and tokens
  const int wr = 64 * (w & 1), wb = 64 * (w >> 1);
  const uint8_t *ss[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    ss[i] = L.ws + (int64_t)min(r0 + wr + 16 * i + c, L.rows - 1) * blocks + 2 * g;
    ss[4 + i] = L.xs + (int64_t)min(b0 + wb + 16 * i + c, L.batch - 1) * blocks + 2 * g;
  }
  // both bytes of a stage's two steps, from the last two where the row has ended (at least two blocks): no
  // load is conditional, what it gives is put right when it is used
  uint16_t sc[8];
  auto scales = [&](int kt) {
    const int b = min(8 * kt, blocks - 2 - 2 * g);
#pragma unroll
    for (int i = 0; i < 8; i++) __builtin_memcpy(&sc[i], ss[i] + b, 2);
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0, 0, 0, 0};
  fill(0);
  scales(0);
  const int swz = (c >> 1) & 7;
  for (int kt = 0; kt < tiles_k; kt++) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int now[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int left = blocks - 8 * kt - 2 * g;  // blocks from this one on
      now[i] = left >= 2 ? (int)sc[i] : (left == 1 ? 0x7f00 | sc[i] >> 8 : 0x7f7f);
    }
    if (kt + 1 < tiles_k) {
      fill(kt + 1);
      scales(kt + 1);
    }
    const uint8_t(*rows)[128] = stage[kt & 1];
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int at = ((2 * g + s) ^ swz) * 16;
      i32x4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        a[i] = *(const i32x4*)&rows[wr + 16 * i + c][at];
        b[i] = *(const i32x4*)&rows[128 + wb + 16 * i + c][at];
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          acc[i][j] = s ? mx_step<1>(a[i], now[i], b[j], now[4 + j], acc[i][j]) : mx_step<0>(a[i], now[i], b[j], now[4 + j], acc[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int tok = b0 + wb + 16 * j + c;
    if (tok >= L.batch) continue;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = r0 + wr + 16 * i + 4 * g;
      if (r < L.rows) mx_out<T>(L.y, tok * L.ldy + r, L.rows - r, wide, acc[i][j]);
    }
  }
}

// The same on stages of one step of 128 columns (four steps a row at least): 64 bytes a row, 16 KiB;
// while one is multiplied the others are on their way. Chunk c of row r lies at c ^ (r / 4 & 3).
// The scale bytes come for four steps at a time (by the step they would be as many requests to
// L2 as the values) and go to registers so: WHOLE where each row's 16 are an aligned 16-byte piece
// (multiples of 512 columns), else the two aligned pieces that hold them are fetched, the second only
// where the row reaches into it. Two workgroups a CU: with the first four stages fit, else three.
//
// A workgroup takes tile after tile; the stages run on from one to the next, so that the next
// tile's are on their way while this one's outputs are written, and a CU's two workgroups drift apart, one
// writing while the other multiplies.
//
// Row 16 (m / 4) + 4 i + m % 4 of a wave's 64 goes to row m of matrix instruction i, so that a lane ends with 16
// neighbouring outputs of a token, P pieces of 16 bytes. P lanes, P tokens, then exchange
// theirs: a store covers all 64 rows of its tokens, 256 or 128 bytes side by side (16384 x 2048 at 2048 tokens
// takes 61 us so, 70 with stores of 64 bytes side by side).
__device__ __forceinline__ int gemm_row(int q) { return (q & ~63) | (q & 12) << 2 | (q >> 4 & 3) << 2 | (q & 3); }

template <typename T>
__device__ __forceinline__ void mx_pack(f32x4 a, f32x4 b, f32x4 c, f32x4 d, u32x4* o) {
  if constexpr (sizeof(T) == 4) {
    o[0] = __builtin_bit_cast(u32x4, a), o[1] = __builtin_bit_cast(u32x4, b);
    o[2] = __builtin_bit_cast(u32x4, c), o[3] = __builtin_bit_cast(u32x4, d);
  } else {
    typedef T t8 __attribute__((ext_vector_type(8)));
    o[0] = __builtin_bit_cast(u32x4, t8{(T)a[0], (T)a[1], (T)a[2], (T)a[3], (T)b[0], (T)b[1], (T)b[2], (T)b[3]});
    o[1] = __builtin_bit_cast(u32x4, t8{(T)c[0], (T)c[1], (T)c[2], (T)c[3], (T)d[0], (T)d[1], (T)d[2], (T)d[3]});
  }
}

// Piece k of lane l and piece l % P of lane (l / P) P + k change places.
template <int P>
__device__ __forceinline__ void mx_turn(u32x4* o, int c) {
  auto swap = [](u32x4& x, u32x4& y, bool odd, auto perm) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? x[e] : y[e]), perm.value, 0xf, 0xf, true);
      x[e] = odd ? got : x[e], y[e] = odd ? y[e] : got;
    }
  };
  const std::integral_constant<int, 0xb1> by1;  // quad lanes 1 0 3 2
  const std::integral_constant<int, 0x4e> by2;  // 2 3 0 1
#pragma unroll
  for (int k = 0; k < P; k += 2) swap(o[k], o[k + 1], c & 1, by1);
  if constexpr (P == 4)
#pragma unroll
    for (int k = 0; k < 2; k++) swap(o[k], o[k + 2], c & 2, by2);
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256, 2) void mx_gemm128_kernel(MxMatmul L, int row_tiles, int tok_tiles, int wide) {
  constexpr int NS = WHOLE ? 4 : 3, SB = 256 * 64, SP = WHOLE ? 16 : 32;  // stages, bytes of one, scale bytes of a row
  constexpr int P = sizeof(T);  // 16-byte pieces of a lane's outputs for a token
  __shared__ __align__(16) uint8_t stage[NS][SB];
  __shared__ __align__(16) uint8_t scale[2][256][SP];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, steps = (blocks + 3) / 4;
  const GemmRun run = gemm_run(row_tiles * tok_tiles);
  if (run.first >= run.stop) return;

  // ---- the stages: what the next fill takes
  const int chunk = (lane & 3) ^ (lane >> 4), wchunk[2] = {(lane & 3) ^ (2 * w & 3), (lane & 3) ^ (2 * w & 3) ^ 1};
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&stage[0][0]);
  const uint32_t sbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&scale[0][0][0]);
  const uint8_t* src[4];
  uintptr_t sfrom[2], send[2];  // the scale bytes' 16-byte piece, the row's end
  int ft = run.first, fk = 0, filled = 0, groups = 0, fslot = 0;
  auto aim = [&]() {
    const GemmTile tile = gemm_tile(ft, row_tiles, tok_tiles);
    const int r0 = tile.r * kGemmTile, b0 = tile.b * kGemmTile;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int r = 32 * w + 16 * j + (lane >> 2);
      src[j] = L.w + (int64_t)min(r0 + r, L.rows - 1) * blocks * 16 + wchunk[j] * 16;
      src[2 + j] = L.x + (int64_t)min(b0 + r, L.batch - 1) * blocks * 16 + chunk * 16;
      const int q = WHOLE ? 64 * (w & 1) + lane : 64 * (w & 1) + 32 * j + (lane >> 1);
      const uintptr_t s = (uintptr_t)(w < 2 ? L.ws + (int64_t)min(r0 + gemm_row(q), L.rows - 1) * blocks
                                            : L.xs + (int64_t)min(b0 + q, L.batch - 1) * blocks);
      sfrom[j] = s & ~(uintptr_t)15;
      send[j] = s + blocks;
    }
  };
  auto fill = [&]() {
    if (ft >= run.stop) return;
    if ((fk & 3) == 0) {
#pragma unroll
      for (int j = 0; j < (WHOLE ? 1 : 2); j++) {
        const uintptr_t p = sfrom[j] + 4 * fk, next = p + 16;
        mx_dma16((const void*)(!WHOLE && (lane & 1) && next < send[j] ? next : p),
                 sbase + (uint32_t)(groups & 1) * (256 * SP) + (uint32_t)(64 * w + 32 * j) * SP);
      }
      groups++;
    }
    const uint32_t to = base + (uint32_t)fslot * SB;
    fslot = fslot + 1 == NS ? 0 : fslot + 1;
    const bool live = WHOLE || 4 * fk + chunk < blocks;  // chunks behind the last are zeros
#pragma unroll
    for (int j = 0; j < 2; j++) {
      mx_dma16(WHOLE || 4 * fk + wchunk[j] < blocks ? src[j] + fk * 64 : (const uint8_t*)mx_zeros, to + (uint32_t)(32 * w + 16 * j) * 64);
      mx_dma16(live ? src[2 + j] + fk * 64 : (const uint8_t*)mx_zeros, to + (uint32_t)(128 + 32 * w + 16 * j) * 64);
    }
    filled++;
    if (++fk == steps) {
      fk = 0;
      ft += run.step;
      if (ft < run.stop) aim();
    }
  };
  aim();
#pragma unroll
  for (int k = 0; k < NS - 1; k++) fill();

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0, 0, 0, 0};
  const int wr = 64 * (w & 1), wb = 128 + 64 * (w >> 1);
  const int at = (g ^ (c >> 2)) * 16, wrow = wr + 16 * (c >> 2) + (c & 3);
  int done = 0, slot = 0, group = 0, stores = 0;  // steps and groups of four; steps for which the outputs' stores are newer than a stage
  uint32_t sa[4][4], sb[4][4];
  auto wait = [&]() {
    // at least four loads a stage: this one's are there when those of the NS - 2 behind it may be missing,
    // and the outputs' stores that were issued between them
    const int behind = filled - done - 1;
    if (behind < 1)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (behind < NS - 2)
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else if (stores > 0)
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * (NS - 2) + 4 * P) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * (NS - 2)) : "memory");
    stores--;
    // everyone's are there, and the stage before has been read
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  for (int t = run.first; t < run.stop; t += run.step) {
    const GemmTile tile = gemm_tile(t, row_tiles, tok_tiles);
    const int r0 = tile.r * kGemmTile, b0 = tile.b * kGemmTile;
    // where the scale bytes of this lane's rows start in the fetched pieces
    int oa[4], ob[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      oa[i] = (wr + 16 * i + c) * SP + (WHOLE ? 0 : 1) * (int)(((uintptr_t)L.ws + (int64_t)min(r0 + wrow + 4 * i, L.rows - 1) * blocks) & 15);
      ob[i] = (wb + 16 * i + c) * SP + (WHOLE ? 0 : 1) * (int)(((uintptr_t)L.xs + (int64_t)min(b0 + wb - 128 + 16 * i + c, L.batch - 1) * blocks) & 15);
    }
    auto scales = [&](int o, uint32_t* out) {
      const uint32_t* p = (const uint32_t*)(&scale[group & 1][0][0] + (o & ~3));
      if constexpr (WHOLE) {
        const u32x4 d = *(const u32x4*)p;
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = d[e] >> (8 * g);
      } else {
        uint32_t d[5];
#pragma unroll
        for (int e = 0; e < 5; e++) d[e] = p[e];
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = __builtin_amdgcn_alignbyte(d[e + 1], d[e], o & 3) >> (8 * g);
      }
    };
    for (int k = 0; k < steps; k += 4, group++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (!WHOLE && k + e >= steps) break;
        wait();
        if (e == 0)
#pragma unroll
          for (int i = 0; i < 4; i++) scales(oa[i], sa[i]), scales(ob[i], sb[i]);
        if (!WHOLE && 4 * (k + e) + 4 > blocks && 4 * (k + e) + g >= blocks)  // behind the last block: zeros of scale 1
#pragma unroll
          for (int i = 0; i < 4; i++) sa[i][e] = sb[i][e] = 127;
        const uint8_t* st = stage[slot];
        slot = slot + 1 == NS ? 0 : slot + 1;
        i32x4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          a[i] = *(const i32x4*)(st + (wrow + 4 * i) * 64 + at);
          b[i] = *(const i32x4*)(st + (wb + 16 * i + c) * 64 + at);
        }
        // the next loads between the products, whose time hides their addresses: 4096 x 4096 at 4096 tokens
        // takes 75 us so, 78 with them before the reads from LDS
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] = mx_step<0>(a[i], (int)sa[i][e], b[j], (int)sb[j][e], acc[i][j]);
          if (i == 1) {
            __builtin_amdgcn_sched_barrier(0);
            fill();
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        done++;
      }
    }
    const bool inner = wide == 2 && r0 + kGemmTile <= L.rows && b0 + kGemmTile <= L.batch;  // then 4 P stores, no more
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int tok = b0 + wb - 128 + 16 * j + c, r = r0 + wr + 16 * g;
      if (inner) {
        u32x4 o[P];
        mx_pack<T>(acc[0][j], acc[1][j], acc[2][j], acc[3][j], o);
        mx_turn<P>(o, c);
#pragma unroll
        for (int k = 0; k < P; k++)
          __builtin_nontemporal_store(o[k], (u32x4*)((T*)L.y + (int64_t)((tok & ~(P - 1)) + k) * L.ldy + r + 16 / P * (c & (P - 1))));
      } else if (tok < L.batch) {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (r + 4 * i < L.rows) mx_out<T>(L.y, tok * L.ldy + r + 4 * i, L.rows - r - 4 * i, wide, acc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    stores = inner ? NS - 1 : 0;
  }
}

template <typename T>
hipError_t gemm_t(const MxMatmul& L) {
  const int rt = (L.rows + kGemmTile - 1) / kGemmTile, tt = (L.batch + kGemmTile - 1) / kGemmTile;
  // outputs: 16 bytes at once, four values at once, or one by one
  const int wide = ((uintptr_t)L.y & 15) == 0 && L.ldy * sizeof(T) % 16 == 0             ? 2
                   : ((uintptr_t)L.y & (4 * sizeof(T) - 1)) == 0 && L.ldy % 4 == 0 ? 1
                                                                                   : 0;
  const unsigned all = (unsigned)((rt * tt + 7) / 8 * 8);
  const dim3 grid(all < 512 ? all : 512);
  if (L.cols % 512 == 0 && ((uintptr_t)L.ws & 15) == 0 && ((uintptr_t)L.xs & 15) == 0)
    hipLaunchKernelGGL((mx_gemm128_kernel<T, true>), grid, dim3(256), 0, L.stream, L, rt, tt, wide);
  else if (L.cols > 384)  // four steps
    hipLaunchKernelGGL((mx_gemm128_kernel<T, false>), grid, dim3(256), 0, L.stream, L, rt, tt, wide);
  else
    hipLaunchKernelGGL((mx_gemm_kernel<T>), dim3(all), dim3(256), 0, L.stream, L, rt, tt, wide);
  return hipGetLastError();
}

}  // namespace

// At least two blocks a row (the scale bytes come in pairs).
hipError_t launch_mx_gemm(const MxMatmul& L) {
  if (L.dtype == kF32) return gemm_t<float>(L);
  return L.dtype == kF16 ? gemm_t<_Float16>(L) : gemm_t<__bf16>(L);
}

}  // namespace nrq
