// Internal interface of the paged INT4 KV-cache kernels (not part of the
// public C ABI; the extern "C" wrappers live in abi.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "spectra_b200.h"

namespace spectra {

constexpr int kTileTokens = 16;  // tokens of one tile of the cache

// Byte offsets inside a tile: 16 tokens of one head, D = 32 G features.
struct TileLayout {
  int G;
  __host__ __device__ constexpr int bytes() const { return 608 * G; }
  __host__ __device__ constexpr int block() const { return 128 * G; }  // codes of 8 tokens
  __host__ __device__ constexpr int k_codes() const { return 0; }
  __host__ __device__ constexpr int v_codes() const { return 256 * G; }
  __host__ __device__ constexpr int k_scales() const { return 512 * G; }
  __host__ __device__ constexpr int v_scales() const { return 544 * G; }
  __host__ __device__ constexpr int k_zeros() const { return 576 * G; }
  __host__ __device__ constexpr int v_zeros() const { return 592 * G; }
};

// A cache and the batch of sequences that a call works on, as the kernels see them.
struct PagedView {
  uint8_t* pool;             // [pages, kv_heads, page / 16, tile]
  int64_t page_stride;       // bytes
  int num_pages, kv_heads, head_dim;
  int page_log2;             // page = 1 << page_log2 tokens
  const int* tables;         // [batch, width] page numbers
  int64_t table_stride;      // elements
  const int* seq_lens;       // [batch] tokens held, the new ones included
  const int* cu_q;           // [batch + 1], or NULL: every sequence has q_len new tokens
  int batch, q_len;
  int64_t total;             // new tokens of the batch
  int max_q;                 // most new tokens of one sequence (the host's bound: the attention keeps to it)
  int limit;                 // positions past this are not touched: min(max_len, width * page)
};

struct PagedAppendArgs {
  PagedView c;
  const void* q; int64_t q_ts, q_hs;       // [total, q_heads, D] or NULL
  void* q_out; int64_t qo_ts, qo_hs;
  const void* k; int64_t k_ts, k_hs;       // [total, kv_heads, D]
  const void* v; int64_t v_ts, v_hs;
  int dtype, q_heads;
  const float* cos; const float* sin; int64_t cs_rs;  // [limit, rotary / 2] or NULL
  int rotary, interleaved;
  int vec;                                 // every row starts on a 16-byte boundary
  int tokens;                              // of a block (set by the launcher)
};
int launch_paged_append(const PagedAppendArgs& a, cudaStream_t st);

struct PagedReadArgs {
  PagedView c;
  void* k; void* v;                        // [total, kv_heads, D], contiguous
  int out_dtype;
  int tokens;                              // of a block (set by the launcher)
};
int launch_paged_read(const PagedReadArgs& a, cudaStream_t st);

struct PagedAttnArgs {
  PagedView c;
  const void* q; int64_t q_ts, q_hs;       // [total, q_heads, D]
  void* out; int64_t o_ts, o_hs;
  int dtype, q_heads, group;               // group = q_heads / kv_heads
  float scale, softcap;                    // softcap 0: none (1e30 at most, which no score feels)
  const float* slopes;                     // [q_heads] or NULL
  int causal, window;                      // window 0: none
  int vec;                                 // rows of q and out on 16-byte boundaries
  void* workspace; size_t workspace_bytes;
};
// A workspace: kPagedCounterBytes of counters (zero between calls), then partial results.
constexpr size_t kPagedCounterBytes = SPECTRA_PAGED_COUNTER_BYTES;
// One or a few tokens per sequence (paged_attn.cu); many (paged_prompt.cu).
// Sequences with more than max_rows (the first) or at most min_rows (the
// second) rows per key/value head are left to the other.
size_t paged_attn_workspace_bytes(int head_dim);
size_t paged_prompt_workspace_bytes(int head_dim);
int launch_paged_attn(const PagedAttnArgs& a, int max_rows, cudaStream_t st);
int launch_paged_prompt(const PagedAttnArgs& a, int min_rows, cudaStream_t st);
int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st);  // the one or the other, or both
int paged_attn_timeouts(long long* out, bool reset);
int paged_prompt_timeouts(long long* out, bool reset);

}  // namespace spectra
