// The MXFP4 product over many tokens: tiles of 128 rows of w by 128 tokens.
//
// A stage holds 256 columns (128 bytes) of the tile's 128 + 128 rows, 32 KiB; two
// stages take turns, filled by direct loads to LDS while the other is
// multiplied, two workgroups a CU. 16-byte chunk c of row r lies at c ^ (r / 2 & 7): the 16
// rows that a matrix instruction's quarter reads at one chunk fall on 16 different
// places of the 64 banks. A wave multiplies 64 rows by 64 tokens; of lane l's
// two steps in a stage, step s takes block 2 (l / 16) + s, so that both scale bytes of a
// row come as one 16-bit load and the instruction picks the byte. Chunks behind
// the last column come from zeros; rows behind the last are the last once more and are not stored.
#include "nrq_serve_launch.h"

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

// The same for whole steps of 128 columns (at least four): four stages of one step each (64 bytes a
// row, 16 KiB), three of them on their way while the fourth is multiplied. Chunk c
// of row r lies at c ^ (r / 4 & 3). The scale bytes come for four steps at a time, 16
// bytes of a row in one piece (by the step they would be as many requests to L2 as the values), and go
// to registers so.
//
// A workgroup takes tile after tile; the stages run on from one to the next, so that the next
// tile's are on their way while this one's outputs are written, and a CU's two workgroups drift apart, one
// writing while the other multiplies.
template <typename T>
__global__ __launch_bounds__(256, 2) void mx_gemm128_kernel(MxMatmul L, int row_tiles, int tok_tiles, int wide) {
  constexpr int NS = 4, SB = 256 * 64;
  __shared__ __align__(16) uint8_t stage[NS][SB];
  __shared__ __align__(16) uint8_t scale[2][256][16];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int blocks = L.cols / 32, steps = blocks / 4;
  const GemmRun run = gemm_run(row_tiles * tok_tiles);
  if (run.first >= run.stop) return;

  // ---- the stages: what the next fill takes
  const int chunk = (lane & 3) ^ (lane >> 4);
  const uint32_t base = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&stage[0][0]);
  const uint32_t sbase = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)&scale[0][0][0]);
  const uint8_t* src[5];
  int ft = run.first, fk = 0, filled = 0, groups = 0;
  auto aim = [&]() {
    const GemmTile tile = gemm_tile(ft, row_tiles, tok_tiles);
    const int r0 = tile.r * kGemmTile, b0 = tile.b * kGemmTile;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int r = 32 * w + 16 * j + (lane >> 2);
      src[j] = L.w + (int64_t)min(r0 + r, L.rows - 1) * blocks * 16 + chunk * 16;
      src[2 + j] = L.x + (int64_t)min(b0 + r, L.batch - 1) * blocks * 16 + chunk * 16;
    }
    const int r = 64 * (w & 1) + lane;
    src[4] = w < 2 ? L.ws + (int64_t)min(r0 + r, L.rows - 1) * blocks : L.xs + (int64_t)min(b0 + r, L.batch - 1) * blocks;
  };
  auto fill = [&]() {
    if (ft >= run.stop) return;
    if ((fk & 3) == 0) {
      // the last 16 of the row where fewer are left
      mx_dma16(src[4] + min(4 * fk, blocks - 16), sbase + (uint32_t)(groups & 1) * 4096 + (uint32_t)w * 1024);
      groups++;
    }
    const uint32_t to = base + (uint32_t)(filled & (NS - 1)) * SB;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      mx_dma16(src[j] + fk * 64, to + (uint32_t)(32 * w + 16 * j) * 64);
      mx_dma16(src[2 + j] + fk * 64, to + (uint32_t)(128 + 32 * w + 16 * j) * 64);
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
  const int at = (g ^ (c >> 2)) * 16;
  int done = 0, group = 0, stores = 0;  // steps and groups of four; steps for which 16 stores are newer than a stage
  uint32_t sa[4][4], sb[4][4];
  auto wait = [&]() {
    // at least four loads a stage: this one's are there when those of the two behind it may be missing, and
    // the outputs' stores that were issued between them
    const int behind = filled - done - 1;
    if (behind < 1)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if (behind < 2)
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else if (stores > 0)
      asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    stores--;
    // everyone's are there, and the stage before has been read
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    fill();
  };
  auto multiply = [&](const uint32_t* va, const uint32_t* vb) {
    const uint8_t* st = stage[done & (NS - 1)];
    i32x4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      a[i] = *(const i32x4*)(st + (wr + 16 * i + c) * 64 + at);
      b[i] = *(const i32x4*)(st + (wb + 16 * i + c) * 64 + at);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) acc[i][j] = mx_step<0>(a[i], (int)va[i], b[j], (int)vb[j], acc[i][j]);
    done++;
  };
  for (int t = run.first; t < run.stop; t += run.step) {
    const GemmTile tile = gemm_tile(t, row_tiles, tok_tiles);
    const int r0 = tile.r * kGemmTile, b0 = tile.b * kGemmTile;
    int k = 0;
    for (; k + 4 <= steps; k += 4) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        wait();
        if (e == 0) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            *(u32x4*)sa[i] = *(const u32x4*)scale[group & 1][wr + 16 * i + c];
            *(u32x4*)sb[i] = *(const u32x4*)scale[group & 1][wb + 16 * i + c];
          }
        }
        uint32_t va[4], vb[4];
#pragma unroll
        for (int i = 0; i < 4; i++) va[i] = sa[i][e] >> (8 * g), vb[i] = sb[i][e] >> (8 * g);
        multiply(va, vb);
      }
      group++;
    }
    if (k < steps) {
      const uint8_t* sc = &scale[group & 1][0][16 - 4 * (steps - k) + g];  // the last 16 bytes of the row
      for (; k < steps; k++, sc += 4) {
        wait();
        uint32_t va[4], vb[4];
#pragma unroll
        for (int i = 0; i < 4; i++) va[i] = sc[(wr + 16 * i + c) * 16], vb[i] = sc[(wb + 16 * i + c) * 16];
        multiply(va, vb);
      }
      group++;
    }
    const bool inner = wide && r0 + kGemmTile <= L.rows && b0 + kGemmTile <= L.batch;  // then 16 stores, no more
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int tok = b0 + wb - 128 + 16 * j + c, r = r0 + wr + 4 * g;
      if (inner) {
#pragma unroll
        for (int i = 0; i < 4; i++) mx_put<T>(L.y, tok * L.ldy + r + 16 * i, acc[i][j]);
      } else if (tok < L.batch) {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (r + 16 * i < L.rows) mx_out<T>(L.y, tok * L.ldy + r + 16 * i, L.rows - r - 16 * i, wide, acc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    stores = inner ? 3 : 0;
  }
}

template <typename T>
hipError_t gemm_t(const MxMatmul& L) {
  const int rt = (L.rows + kGemmTile - 1) / kGemmTile, tt = (L.batch + kGemmTile - 1) / kGemmTile;
  const int wide = ((uintptr_t)L.y & (4 * sizeof(T) - 1)) == 0 && L.ldy % 4 == 0;
  const unsigned all = (unsigned)((rt * tt + 7) / 8 * 8);
  const bool steps = L.cols % 128 == 0 && L.cols >= 512 && ((uintptr_t)L.ws & 3) == 0 && ((uintptr_t)L.xs & 3) == 0;
  if (steps)
    hipLaunchKernelGGL((mx_gemm128_kernel<T>), dim3(all < 512 ? all : 512), dim3(256), 0, L.stream, L, rt, tt, wide);
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
