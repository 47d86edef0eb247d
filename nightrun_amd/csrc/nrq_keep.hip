// The move of an accepted path's keys and values (include/nrq_tree.h, nrq_dev_keep_path).
//
// A thread owns 8 dimensions of one head of one layer's keys or values and takes the path's nodes in order: a node never
// comes from before its place, so what it loads has not been written over by the nodes before it, and nobody else touches
// it. Every wave reads the path for itself, lane i looks up both places of its entry i. A few moves of 16 bytes
// a thread: a launch and a chain of dependent loads (length and path, page, values) bound it. What one chat accepted, 16 layers of
// 8 heads of 64, takes 1.9 us behind other work and 6.6 called from Python; 48 chats, heads of 128, 8.5.
#include "nrq_page.h"
#include "nrq_tree_launch.h"

namespace nrq {
namespace {

constexpr int kKeepNT = 256;
constexpr int kKeepAhead = 8;  // moves of a thread on their way together

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kKeepNT) void keep_path_kernel(KeepLaunch L, int seq0, int chunks, int items) {
  const int b = seq0 + blockIdx.y, lane = threadIdx.x & 63;
  const int64_t held = (int64_t)L.table.width * L.kv.page_size;
  const int len = (int)min((int64_t)max(L.lens[b], 0), held);
  const int n = L.counts ? min(max(L.counts[b], 0), L.n_new) : L.n_new, base = len - n;
  const int from = lane < n ? L.path[(int64_t)b * L.n_new + lane] : -1, before = __shfl_up(from, 1);
  const unsigned long long bad = ~__ballot(from >= 0 && from < n && (lane == 0 || from > before));
  const int kept = bad ? __ffsll(bad) - 1 : 64;
  if (blockIdx.x == 0 && threadIdx.x == 0) L.new_lens[b] = max(base + kept, 0);
  uint32_t src = kNoPlace, dst = kNoPlace;
  if (lane < kept && from != lane) {
    const int* pages = L.table.pages + b * L.table.stride;
    src = page_place(pages, L.table.width, L.kv.page_size, L.kv.n_pages, L.kv.page_stride8, L.kv.pos_stride8, base + from);
    dst = page_place(pages, L.table.width, L.kv.page_size, L.kv.n_pages, L.kv.page_stride8, L.kv.pos_stride8, base + lane);
  }
  const unsigned long long moves = __ballot(src != kNoPlace && dst != kNoPlace);
  const int i = blockIdx.x * kKeepNT + threadIdx.x;
  const bool on = i < items;
  const int j = on ? i : 0, c = j % chunks, r = j / chunks, v = r & 1, h = (r >> 1) % L.kv.n_kv, layer = (r >> 1) / L.kv.n_kv;
  uint16_t* pool = (v ? L.kv.v : L.kv.k) + layer * L.layer_stride + h * L.kv.head_stride + 8 * c;
  const int some = min(8, L.kv.hd - 8 * c);  // dimensions
  for (unsigned long long m = moves; m;) {
    u32x4 x[kKeepAhead];
    uint32_t to[kKeepAhead];
    unsigned long long left = m;
#pragma unroll
    for (int k = 0; k < kKeepAhead; k++) {
      to[k] = kNoPlace;
      if (!left) continue;
      const int e = __ffsll(left) - 1;
      left &= left - 1;
      const uint16_t* p = pool + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)src, e) * 8;
      to[k] = __builtin_amdgcn_readlane((int)dst, e);
      if (!on) continue;
      if (some == 8)
        x[k] = *(const u32x4*)p;
      else
#pragma unroll
        for (int d = 0; d < 7; d++)
          if (d < some) x[k][d / 2] = d & 1 ? x[k][d / 2] | (uint32_t)p[d] << 16 : p[d];
    }
#pragma unroll
    for (int k = 0; k < kKeepAhead; k++) {
      if (to[k] == kNoPlace || !on) continue;
      uint16_t* p = pool + (uint64_t)to[k] * 8;
      if (some == 8)
        *(u32x4*)p = x[k];
      else
#pragma unroll
        for (int d = 0; d < 7; d++)
          if (d < some) p[d] = (uint16_t)(x[k][d / 2] >> (d & 1 ? 16 : 0));
    }
    m = left;
  }
}

}  // namespace

hipError_t launch_keep(const KeepLaunch& L) {
  const int chunks = (L.kv.hd + 7) / 8, items = L.layers * L.kv.n_kv * 2 * chunks;
  const int groups = (items + kKeepNT - 1) / kKeepNT;
  // a grid has fewer than 2^32 threads, and 65535 rows
  const int most = groups >= 1 << 8 ? (1 << 23) / groups : 65535 / 2;
  for (int b0 = 0; b0 < L.table.seqs; b0 += most) {
    const int n = L.table.seqs - b0 < most ? L.table.seqs - b0 : most;
    hipLaunchKernelGGL(keep_path_kernel, dim3(groups > 0 ? groups : 1, n), dim3(kKeepNT), 0, L.stream, L, b0, chunks, items);
  }
  return hipGetLastError();
}

}  // namespace nrq
