// The paged cache's index arithmetic, for kernels and (compiled alone by a host
// compiler) for the tests: where a position lies, what a sequence's new tokens
// see, and how the line of all tiles is cut among workgroups.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define NRQ_HD __host__ __device__ __forceinline__
#else
#define NRQ_HD inline
#endif

namespace nrq {

constexpr uint32_t kNoPlace = 0xffffffffu;

// The place (in units of 8 elements from the pool's start, as the strides are given) of
// position t on the pages of one sequence, kNoPlace where there is none: outside
// the table, or on an entry that is no page.
NRQ_HD uint32_t page_place(const int* pages, int width, int page_size, int n_pages, uint32_t page_stride8,
                           uint32_t pos_stride8, int t) {
  if (t < 0) return kNoPlace;
  const uint32_t p = (uint32_t)t / (uint32_t)page_size;
  if (p >= (uint32_t)width) return kNoPlace;
  const int page = pages[p];
  if (page < 0 || page >= n_pages) return kNoPlace;
  return (uint32_t)page * page_stride8 + ((uint32_t)t - p * (uint32_t)page_size) * pos_stride8;
}

// A sequence of the attention: its positions and new tokens (clamped), the first
// position of its first tile and its tiles (one at least, also for nothing).
struct SeqSpan {
  int len, n, start, tiles;
};
NRQ_HD SeqSpan seq_span(int len, int count, int n_new, int64_t held, int window, int tile) {
  SeqSpan s;
  const int64_t most = held < 0x7fffffff ? held : 0x7fffffff;
  s.n = count < 0 ? 0 : (count > n_new ? n_new : count);
  s.len = len < 0 || s.n == 0 ? 0 : (len > most ? (int)most : len);
  // the first new token is at len - n and sees from len - n + 1 - window
  const int64_t from = (int64_t)s.len - s.n + 1 - window;
  s.start = window > 0 && from > 0 ? (int)from & ~15 : 0;
  const int64_t t = ((int64_t)s.len - s.start + tile - 1) / tile;
  s.tiles = t > 1 ? (int)t : 1;
  return s;
}

// The line of `total` tiles among `wgs` <= total workgroups: the first total % wgs
// take one tile more. line_start(wgs) is total.
NRQ_HD int line_start(int w, int total, int wgs) {
  const int each = total / wgs, more = total - each * wgs;
  return w * each + (w < more ? w : more);
}
// The workgroup that takes tile g.
NRQ_HD int line_owner(int g, int total, int wgs) {
  const int each = total / wgs, more = total - each * wgs, big = more * (each + 1);
  return g < big ? g / (each + 1) : more + (g - big) / each;
}

}  // namespace nrq
