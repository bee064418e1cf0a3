// Device helpers shared by the paged INT4 KV-cache kernels.
#pragma once

#include "common.cuh"
#include "paged.h"

namespace spectra {

// First row and number of rows of a sequence's new tokens.
__device__ __forceinline__ void new_tokens(const PagedView& c, int b, int64_t& first, int& count) {
  if (c.cu_q) {
    const int at = c.cu_q[b], end = c.cu_q[b + 1];
    first = at < 0 ? 0 : at;
    const int64_t last = end < c.total ? int64_t(end) : c.total;
    count = last > first ? int(last - first) : 0;
  } else {
    first = int64_t(b) * c.q_len;
    const int64_t left = c.total - first;
    count = left < c.q_len ? (left > 0 ? int(left) : 0) : c.q_len;
  }
}

// Sequence of new token t, or -1 where none holds it.
__device__ __forceinline__ int sequence_of(const PagedView& c, int64_t t) {
  if (!c.cu_q) {
    const int64_t b = t / c.q_len;
    return b < c.batch ? int(b) : -1;
  }
  int lo = 0, hi = c.batch;  // the last b with cu_q[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  return t >= c.cu_q[lo] && t < c.cu_q[lo + 1] ? lo : -1;
}

// Tile that holds position `pos` (0 <= pos < limit) of head h, or NULL where
// the block table names no page of the pool.
__device__ __forceinline__ uint8_t* tile_of(const PagedView& c, int b, int h, int pos) {
  const int page = c.tables[b * c.table_stride + (pos >> c.page_log2)];
  if (unsigned(page) >= unsigned(c.num_pages)) return nullptr;
  const int tiles = 1 << (c.page_log2 - 4);
  const int tile = (pos >> 4) & (tiles - 1);
  const TileLayout L{c.head_dim / 32};
  return c.pool + page * c.page_stride + (int64_t(h) * tiles + tile) * L.bytes();
}

}  // namespace spectra
