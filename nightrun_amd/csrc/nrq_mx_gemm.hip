// The MXFP4 product over many tokens: tiles of 128 rows of w by 128 tokens, or 256 by 256.
//
// y[b][r] = sum over blocks k of 2^(es + et - 254) * sum over the block's 32 columns of the E2M1
// products, summed in 32 bits by the scaled matrix instruction (16 x 16 x 128, a scale byte per row and
// block); rounded once, at the store. 2048 f32 tokens by 16384 x 2048, their quantization included, take
// 60 us: 2.3 PFLOP/s and 2.2 TB/s of f32 outputs; 2048 tokens by 8192 x 8192 95 us, 2.9 PFLOP/s (7.1 come out
// of registers). What bounds it is the way of the values from L2 over LDS to the registers (a tile of 128 takes 256 products
// a byte, one of 256 takes 512), and at few columns the outputs: of the 111,000 clocks of the first, a CU's LDS is read for
// 41,000 and filled for 16,000, 16,000 go to bank conflicts, and its matrix units work for 33,000.
//
// Up to 384 columns (and beyond 2^26) one kernel takes a tile a workgroup, in steps of 256 columns; else
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
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0), "v"(g) : "memory");
}

// the same from `at` bytes behind a wave-uniform address
__device__ __forceinline__ void mx_dma16(const uint8_t* g, uint32_t at, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(m0), "v"(at), "s"(g) : "memory");
}

template <int S>
__device__ __forceinline__ f32x4 mx_step(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  const i32x8 x = {a.x, a.y, a.z, a.w, 0, 0, 0, 0}, y = {b.x, b.y, b.z, b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, S, sa, S, sb);
}

// the same by the byte, after unrolling a constant
__device__ __forceinline__ f32x4 mx_steps(int s, i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  return s == 0 ? mx_step<0>(a, sa, b, sb, c) : s == 1 ? mx_step<1>(a, sa, b, sb, c) : s == 2 ? mx_step<2>(a, sa, b, sb, c) : mx_step<3>(a, sa, b, sb, c);
}

// 16 bytes of outputs past the caches, which w and the tokens fill: 16384 x 2048 at 2048 tokens takes 60.5 us so, 62.8
// through them, 8192 tokens 228 and 243; f32 outputs that the last-level cache holds go faster through it behind long
// sums (4096 x 4096 at 4096 tokens 59.5, past it 63.6), 16-bit ones the same. Rows need not be aligned.
template <typename T>
__device__ __forceinline__ void mx_put(T* y, u32x4 v) {
  typedef u32x4 any __attribute__((aligned(2)));
  __builtin_nontemporal_store(v, (any*)y);
}

// the same where the row has n left
template <typename T>
__device__ __forceinline__ void mx_some(T* y, int n, u32x4 v) {
  constexpr int E = 16 / sizeof(T);
  typedef T te __attribute__((ext_vector_type(E)));
  if (n >= E) return mx_put(y, v);
  const te o = __builtin_bit_cast(te, v);
#pragma unroll
  for (int i = 0; i < E - 1; i++)
    if (i < n) y[i] = o[i];
}

template <typename T>
__device__ __forceinline__ void mx_out(void* y, int64_t at, int n, bool wide, f32x4 v) {
  if (wide && n >= 4) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    __builtin_nontemporal_store(o, (t4*)((T*)y + at));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) ((T*)y)[at + i] = (T)v[i];
  }
}

// Workgroups go round the eight XCDs; each XCD gets a run of the tiles, of which its workgroups
// take every step-th. Tiles go by groups of up to 16 row tiles, within a group by tokens, and for the
// same tokens by rows: so an XCD keeps its rows of w in its L2, and what it writes at a
// time lies together (by tokens first, 16384 x 2080 at 2048 tokens takes 77 us, so 72).
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

// The same on stages of one step of 128 columns (four steps a row at least), 64 bytes a row;
// while one is multiplied the others are on their way. Chunk c of row r lies at c ^ (r / 4 & 3), of a row
// of w at c ^ (r / 16 & 3). A wave multiplies 64 rows by TILE / 2 tokens.
// The scale bytes come for four steps at a time (by the step they would be as many requests to
// L2 as the values), and a lane keeps its four of a row in one register: WHOLE where each row's 16 are an
// aligned 16-byte piece (multiples of 512 columns), else the two aligned pieces that hold them are
// fetched, the second only where the row reaches into it. With tiles of 128 two workgroups share a CU:
// in the first case four stages fit, else three.
//
// A workgroup takes tile after tile; the stages run on from one to the next, so that the next
// tile's are on their way while this one's outputs are written; a CU's two workgroups drift apart, one
// writing while the other multiplies.
//
// Row 16 (m / 4) + 4 i + m % 4 of a wave's 64 goes to row m of matrix instruction i, so that a lane ends with 16
// neighbouring outputs of a token, P pieces of 16 bytes. P lanes, P tokens, then exchange
// theirs: a store covers all 64 rows of its tokens, 256 or 128 bytes side by side (16384 x 2048 at 2048 tokens
// takes 61 us so, 70 with stores of 64 bytes side by side). Rows of any alignment are stored so: 16385 x 2048 at 3000
// tokens takes 100 us, 172 with a store for each value that is not aligned.
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

// Part p of `parts` of a row's steps starts here: whole groups of four, the rest with the last.
__device__ __forceinline__ int gemm_part(int p, int parts, int steps) {
  return p == parts ? steps : __builtin_amdgcn_readfirstlane(4 * ((steps >> 2) * p / parts));
}

template <typename T, bool WHOLE, int TILE, bool PARTS>
__global__ __launch_bounds__(2 * TILE, 2) void mx_gemm128_kernel(MxMatmul L, int row_tiles, int tok_tiles, int parts, int64_t plane) {
  constexpr int NS = WHOLE ? 4 : 3, ROWS = 2 * TILE, SB = ROWS * 64, SP = WHOLE ? 16 : 32;  // stages, bytes of one, scale bytes of a row
  constexpr int HALF = TILE / 64, JT = TILE / 32;  // waves to a half of the tile's rows or tokens, products of a wave along the tokens
  constexpr int P = sizeof(T), E = 16 / sizeof(T);  // 16-byte pieces of a lane's outputs for a token, values of one
  __shared__ __align__(16) uint8_t stage[NS][SB];
  __shared__ __align__(16) uint8_t scale[2][ROWS][SP];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, steps = (blocks + 3) / 4;
  const int tiles = row_tiles * tok_tiles;
  const GemmRun run = gemm_run(PARTS ? tiles * parts : tiles);
  if (run.first >= run.stop) return;

  // ---- the stages: what the next fill takes
  const bool of_w = w < HALF;  // whose 64 rows this wave fetches, every quarter of them (w) or row (tokens) its own order of chunks
  int chunk[4];
#pragma unroll
  for (int j = 0; j < 4; j++) chunk[j] = (lane & 3) ^ (of_w ? j : lane >> 4);
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&stage[0][0]);
  const uint32_t sbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&scale[0][0][0]);
  const uint32_t row = (uint32_t)blocks * 16;
  const uint8_t *values, *sbytes;  // of the wave's first row; sbytes down to a multiple of 16
  uint32_t src[4], sfrom[2], send[2];  // from there: chunks of step 0; a row's first 16-byte piece of scales, its end
  int ft = run.first, fk = 0, fstop = 0, filled = 0, groups = 0, fslot = 0;
  auto aim = [&]() {
    const int part = PARTS ? __builtin_amdgcn_readfirstlane(ft / tiles) : 0;
    fk = PARTS ? gemm_part(part, parts, steps) : 0;
    fstop = PARTS ? gemm_part(part + 1, parts, steps) : steps;
    const GemmTile tile = gemm_tile(ft - part * tiles, row_tiles, tok_tiles);
    const int first = of_w ? tile.r * TILE + 64 * w : tile.b * TILE + 64 * (w - HALF), all = of_w ? L.rows : L.batch;
    const int from = min(first, all - 1), last = all - 1 - from;
    const uintptr_t s = (uintptr_t)(of_w ? L.ws : L.xs) + (int64_t)from * blocks;
    values = (of_w ? L.w : L.x) + (int64_t)from * row;
    sbytes = (const uint8_t*)(s & ~(uintptr_t)15);
#pragma unroll
    for (int j = 0; j < 4; j++) src[j] = min(16 * j + (lane >> 2), last) * row + chunk[j] * 16;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int q = WHOLE ? lane : 32 * j + (lane >> 1);
      const uint32_t at = (uint32_t)(s & 15) + min(of_w ? gemm_row(q) : q, last) * blocks;
      sfrom[j] = at & ~15u;
      send[j] = at + blocks;
    }
  };
  auto fill = [&]() {
    if (ft >= run.stop) return;
    if ((fk & 3) == 0) {
#pragma unroll
      for (int j = 0; j < (WHOLE ? 1 : 2); j++) {
        const uint32_t p = sfrom[j] + 4 * fk, next = p + 16;
        mx_dma16(sbytes, !WHOLE && (lane & 1) && next < send[j] ? next : p,
                 sbase + (uint32_t)(groups & 1) * (ROWS * SP) + (uint32_t)(64 * w + 32 * j) * SP);
      }
      groups++;
    }
    const uint32_t to = base + (uint32_t)fslot * SB + (uint32_t)w * 4096;
    fslot = fslot + 1 == NS ? 0 : fslot + 1;
#pragma unroll
    for (int j = 0; j < 4; j++)  // in place of chunks behind the last the step's first, cleared when used
      mx_dma16(values + fk * 64, WHOLE || 4 * fk + chunk[j] < blocks ? src[j] : src[j] - chunk[j] * 16, to + j * 1024);
    filled++;
    if (++fk == fstop) {
      ft += run.step;
      if (ft < run.stop) aim();
    }
  };
  aim();
#pragma unroll
  for (int k = 0; k < NS - 1; k++) fill();

  f32x4 acc[4][JT];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < JT; j++) acc[i][j] = f32x4{0, 0, 0, 0};
  const int wr = 64 * (w & (HALF - 1)), wb = TILE + TILE / 2 * (w / HALF);
  const int at = (g ^ (c >> 2)) * 16, wrow = wr + 16 * (c >> 2) + (c & 3);
  int done = 0, slot = 0, group = 0, stores = 0;  // steps and groups of four; steps for which the outputs' stores are newer than a stage
  uint32_t sa[4], sb[JT];  // of a row: byte e for step e
  const uint32_t pick = 0x0c0c0400u + 0x0101u * g;  // byte g of two words to the low half
  auto wait = [&]() {
    // at least four loads a stage: this one's are there when those of the NS - 2 behind it may be missing,
    // and the outputs' stores that were issued between them
    const int behind = filled - done - 1;
    if (behind < 1)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (behind < NS - 2)
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else if (stores > 0)
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * (NS - 2) + JT * P) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(4 * (NS - 2)) : "memory");
    stores--;
    // everyone's are there, and the stage before has been read
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  for (int t = run.first; t < run.stop; t += run.step) {
    const int part = PARTS ? __builtin_amdgcn_readfirstlane(t / tiles) : 0;
    const int from = PARTS ? gemm_part(part, parts, steps) : 0, to_step = PARTS ? gemm_part(part + 1, parts, steps) : steps;
    const GemmTile tile = gemm_tile(t - part * tiles, row_tiles, tok_tiles);
    const int r0 = tile.r * TILE, b0 = tile.b * TILE;
    // where the scale bytes of this lane's rows start in the fetched pieces
    int oa[4], ob[JT];
#pragma unroll
    for (int i = 0; i < 4; i++)
      oa[i] = (wr + 16 * i + c) * SP + (WHOLE ? 0 : (int)(((uintptr_t)L.ws + (int64_t)min(r0 + wrow + 4 * i, L.rows - 1) * blocks) & 15));
#pragma unroll
    for (int j = 0; j < JT; j++)
      ob[j] = (wb + 16 * j + c) * SP + (WHOLE ? 0 : (int)(((uintptr_t)L.xs + (int64_t)min(b0 + wb - TILE + 16 * j + c, L.batch - 1) * blocks) & 15));
    auto scales = [&](int o) {
      const uint32_t* p = (const uint32_t*)(&scale[group & 1][0][0] + (o & ~3));
      u32x4 d;
      if constexpr (WHOLE) {
        d = *(const u32x4*)p;
      } else {
        uint32_t f[5];
#pragma unroll
        for (int e = 0; e < 5; e++) f[e] = p[e];
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = __builtin_amdgcn_alignbyte(f[e + 1], f[e], o & 3);
      }
      return __builtin_amdgcn_perm(d[1], d[0], pick) | __builtin_amdgcn_perm(d[3], d[2], pick << 16 | pick >> 16);
    };
    for (int k = from; k < to_step; k += 4, group++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (k + e >= to_step) break;
        wait();
        if (e == 0) {
#pragma unroll
          for (int i = 0; i < 4; i++) sa[i] = scales(oa[i]);
#pragma unroll
          for (int j = 0; j < JT; j++) sb[j] = scales(ob[j]);
        }
        const uint8_t* st = stage[slot];
        slot = slot + 1 == NS ? 0 : slot + 1;
        i32x4 a[4], b[JT];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = *(const i32x4*)(st + (wrow + 4 * i) * 64 + at);
#pragma unroll
        for (int j = 0; j < JT; j++) b[j] = *(const i32x4*)(st + (wb + 16 * j + c) * 64 + at);
        if (!WHOLE && 4 * (k + e) + 4 > blocks && 4 * (k + e) + g >= blocks) {  // behind the last block: zeros, scales of 1
#pragma unroll
          for (int i = 0; i < 4; i++) a[i] = i32x4{0, 0, 0, 0}, sa[i] = 0x7f7f7f7f;
#pragma unroll
          for (int j = 0; j < JT; j++) sb[j] = 0x7f7f7f7f;
        }
        // the next loads between the products, whose time hides their addresses: 2560 x 9728 at 4096 tokens
        // takes 111 us so, 114 with them before the reads from LDS
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
          for (int j = 0; j < JT; j++) acc[i][j] = mx_steps(e, a[i], (int)sa[i], b[j], (int)sb[j], acc[i][j]);
          if (i == 1) {
            __builtin_amdgcn_sched_barrier(0);
            fill();
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        done++;
      }
    }
    const bool inner = r0 + TILE <= L.rows && b0 + TILE <= L.batch;  // then JT P stores, no more
#pragma unroll
    for (int j = 0; j < JT; j++) {
      const int tok = (b0 + wb - TILE + 16 * j + c) & ~(P - 1), r = r0 + wr + 16 * g + E * (c & (P - 1));
      u32x4 o[P];
      mx_pack<T>(acc[0][j], acc[1][j], acc[2][j], acc[3][j], o);
      mx_turn<P>(o, c);
      T* to = (T*)L.y + part * plane + (int64_t)tok * L.ldy + r;
#pragma unroll
      for (int k = 0; k < P; k++)
        if (inner)
          mx_put<T>(to + k * L.ldy, o[k]);
        else if (tok + k < L.batch)
          mx_some<T>(to + k * L.ldy, L.rows - r, o[k]);
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    stores = inner ? NS - 1 : 0;
  }
}

// The sums over the parts of the rows, in order: y from the planes, E values a thread.
template <typename T>
__global__ __launch_bounds__(256) void mx_parts_kernel(MxMatmul L, const float* sums, int parts, int64_t plane, int ld) {
  constexpr int E = 16 / sizeof(T);
  const int each = ld / E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, tok = i / each;
  const int r = (int)(i - tok * each) * E;
  if (tok >= L.batch || r >= L.rows) return;
  f32x4 y[E / 4];
#pragma unroll
  for (int h = 0; h < E / 4; h++) y[h] = *(const f32x4*)(sums + tok * ld + r + 4 * h);
#pragma unroll 4
  for (int p = 1; p < parts; p++)
#pragma unroll
    for (int h = 0; h < E / 4; h++) y[h] += *(const f32x4*)(sums + p * plane + tok * ld + r + 4 * h);
  typedef T te __attribute__((ext_vector_type(E)));
  te o;
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = (T)y[e >> 2][e & 3];
  mx_some<T>((T*)L.y + tok * L.ldy + r, L.rows - r, __builtin_bit_cast(u32x4, o));
}

template <typename T, bool WHOLE, int TILE, bool PARTS = false>
hipError_t gemm_run_tiles(const MxMatmul& L, int parts = 1, int64_t plane = 0) {
  const int rt = (L.rows + TILE - 1) / TILE, tt = (L.batch + TILE - 1) / TILE;
  const int all = (rt * tt * parts + 7) / 8 * 8, most = 256 * 256 / TILE;  // as many workgroups as the card holds
  hipLaunchKernelGGL((mx_gemm128_kernel<T, WHOLE, TILE, PARTS>), dim3(all < most ? all : most), dim3(2 * TILE), 0, L.stream, L, rt, tt, parts, plane);
  return hipGetLastError();
}

int gemm_ld(int rows) { return (rows + 7) & ~7; }

// Parts of the rows: where tiles of 128 leave workgroups of the card idle, their steps are shared out, eight or more to
// a part. A step takes a workgroup about 0.42 us; the parts' sums go to memory and back at about 4.5 TB/s, and adding
// them up is a launch of 3 us. 2560 x 9728 by 64, 128 and 512 tokens takes 15, 18 and 29 us in parts, 34, 38 and 41
// in whole rows; 9728 x 2560 by 256, for which two parts would take 24, 15 in whole ones.
int gemm_parts(int rows, int cols, int batch) {
  if (cols <= 384 || cols > 1 << 26) return 1;
  const int64_t tiles = (int64_t)((rows + 127) / 128) * ((batch + 127) / 128);
  const int most = (cols + 127) / 128 / 8;
  if (tiles > 256 || most < 2) return 1;
  const int fit = (int)(512 / tiles), top = fit < most ? fit : most;
  const double whole = 0.42 * ((cols + 127) / 128), plane = (double)rows * batch * 8 / 4.5e6;
  int parts = 1;
  double best = whole;
  for (int p = 2; p <= top; p++)
    if (whole / p + plane * p + 3.0 < best) best = whole / p + plane * p + 3.0, parts = p;
  return parts;
}

// Tiles of 256 where there are columns enough and tiles enough. A round of them (256 tiles) takes 1.7 times as long
// as one of 512 tiles of 128: 2048 x 8192 at 8192 columns takes 95 us on them, 116 on the smaller (one round,
// two), 2560 x 4096 at 9728 112 and 121, but 9728 x 2048 at 2560 59 and 50 (two, three), 2048 x 2048 at 8192 77 and 48 (one,
// one). Up to 2048 columns the outputs weigh as much as the products, which the larger tile's one workgroup a CU
// does not overlap: 16384 x 2048 at 2048 takes 63 us and 61 (at 4096 97 and 114).
static bool gemm_big(const MxMatmul& L) {
  if (L.cols <= 2048) return false;
  const int64_t big = (int64_t)((L.rows + 255) / 256) * ((L.batch + 255) / 256);
  const int64_t small = (int64_t)((L.rows + 127) / 128) * ((L.batch + 127) / 128);
  return 17 * ((big + 255) / 256) <= 10 * ((small + 511) / 512);
}

template <typename T>
hipError_t gemm_t(const MxMatmul& L) {
  if (L.cols <= 384 || L.cols > 1 << 26) {  // beyond, 64 rows pass 32-bit offsets
    const int wide = ((uintptr_t)L.y & (4 * sizeof(T) - 1)) == 0 && L.ldy % 4 == 0;
    const int rt = (L.rows + kGemmTile - 1) / kGemmTile, tt = (L.batch + kGemmTile - 1) / kGemmTile;
    hipLaunchKernelGGL((mx_gemm_kernel<T>), dim3((rt * tt + 7) / 8 * 8), dim3(256), 0, L.stream, L, rt, tt, wide);
    return hipGetLastError();
  }
  const bool whole = L.cols % 512 == 0 && ((uintptr_t)L.ws & 15) == 0 && ((uintptr_t)L.xs & 15) == 0, big = gemm_big(L);
  const int parts = gemm_parts(L.rows, L.cols, L.batch);
  if (parts > 1) {
    MxMatmul S = L;
    S.y = L.workspace, S.ldy = gemm_ld(L.rows);
    const int64_t plane = S.ldy * L.batch;
    if (hipError_t e = whole ? gemm_run_tiles<float, true, 128, true>(S, parts, plane) : gemm_run_tiles<float, false, 128, true>(S, parts, plane)) return e;
    const int64_t items = plane / (16 / (int)sizeof(T));
    hipLaunchKernelGGL((mx_parts_kernel<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, L.stream, L, (const float*)L.workspace, parts, plane, (int)S.ldy);
    return hipGetLastError();
  }
  if (whole) return big ? gemm_run_tiles<T, true, 256>(L) : gemm_run_tiles<T, true, 128>(L);
  return big ? gemm_run_tiles<T, false, 256>(L) : gemm_run_tiles<T, false, 128>(L);
}

}  // namespace

// The kernel of few columns takes a workgroup of 256 threads for each tile, of which a launch takes fewer than 2^24.
bool mx_gemm_fits(int rows, int cols, int batch) {
  return (cols > 384 && cols <= 1 << 26) || (int64_t)((rows + 127) / 128) * ((batch + 127) / 128) <= (1 << 24) - 8;
}

size_t mx_gemm_workspace(int rows, int cols, int batch) {
  const int parts = gemm_parts(rows, cols, batch);
  return parts > 1 ? (size_t)parts * batch * gemm_ld(rows) * sizeof(float) : 0;
}

// At least two blocks a row (the scale bytes come in pairs).
hipError_t launch_mx_gemm(const MxMatmul& L) {
  if (L.dtype == kF32) return gemm_t<float>(L);
  return L.dtype == kF16 ? gemm_t<_Float16>(L) : gemm_t<__bf16>(L);
}

}  // namespace nrq
