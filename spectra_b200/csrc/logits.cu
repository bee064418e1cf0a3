// Rules on a step's logits and the greedy choice under them, for sm_100a.
//
// For token v of row m, in fp32, every step rounded by itself:
//   v in ids[0 .. len):  x = x > 0 ? x / r : x r
//   n = times of v in ids[prompt .. len), n > 0:  x = (x - f n) - p
//   x = x + b(v),  b of the last entry that names v
//   v not allowed:  x = -inf
// and the token: first maximum of x among the allowed (NaN above every number).
//
// Logits move in units of 16 bytes cut at 16-byte addresses (rows of an odd
// vocabulary start anywhere), as pairs of 16 bits where they lie so.  Two ways:
//
// Few rows: one kernel, a row to a cluster of 1 to 8 CTAs, which take its 128
// bytes by turns (the frequent tokens of a vocabulary lie together).  A CTA has
// a word of shared memory per token, which counts: 19 bits the token's ids, one
// says that the prompt holds it, 12 name its bias.  Whole numbers are added up
// (atomics in shared memory), so their order does not matter, and a list costs
// one pass over it whatever the vocabulary.  The words that are not 0 are
// listed.  Then a thread for each token met replaces its word by the new logit;
// a pass over the row writes what may follow and was not met as it is, and
// -infinity elsewhere; a thread for each token met writes its logit over it.
// (Rules applied in the pass over the row took twice as long: some lane of every
// warp has a rule.)
//
// Many rows: the pass over the rows by a kernel of its own, light enough to fill
// the GPU, which masks and finds the maximum of every 1024 columns (fp32: 512); and a CTA per
// row that counts in a table of the tokens met (the same words, found by their
// token), while that pass is still running, then writes their logits and puts
// the maxima together.  Columns whose maximum was met are looked through again
// without the tokens met.
//
// Measured (with the choice): one row of 128256, 1281 ids, 7.7 us; 64 rows, up to
// 8192 ids, 300 biases and masks, 28.8 us (0.18 of the copy rate: issue slots half
// taken by list look-ups and address arithmetic, and phases that wait for one
// another); 333 rows of 50001, 30.8 us; masks alone, 64 rows 8.6 us (0.6).
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "gemv_mma.cuh"
#include "logits.h"
#include "sm100_ptx.cuh"

namespace spectra {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;                  // CTAs per row, a power of two (8: a portable cluster size)
constexpr int kUnits = 4;                       // 16-byte units that a thread takes in a chunk
constexpr int kFlight = 8;                      // ids of a thread in flight
constexpr uint32_t kCountBits = 19, kPrompt = 1u << kCountBits, kSlot = kCountBits + 1;
constexpr uint32_t kCountMask = kPrompt - 1, kLow = (1u << kSlot) - 1;
static_assert(SPECTRA_MAX_RULE_IDS <= kCountMask && SPECTRA_MAX_RULE_BIASES < (1 << (32 - kSlot)), "a word's fields");

template <int DT>
constexpr int kPer = DT == SPECTRA_DT_F32 ? 4 : 8;  // logits of a unit
template <int DT>
constexpr int kChunk = kThreads * kUnits * kPer<DT>;  // columns that a CTA takes at once
constexpr int kTurn = 3;                              // log2 of the units that a CTA takes before it is the next one's turn

__device__ __forceinline__ int clamp_len(int v, int64_t most) { return v < 0 ? 0 : (v < most ? v : int(most)); }

// The order of a choice as whole numbers: larger value first, a NaN above every number; 0: none.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return ~0u;
  const uint32_t u = __float_as_uint(v + 0.f);  // (-0 as 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == ~0u) return __uint_as_float(0x7FFFFFFFu);
  return o == 0 ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
struct Choice {
  uint32_t order;
  int column;
};
// The best of the warp's, in every lane: the first of the highest.
__device__ __forceinline__ Choice best_of_warp(const Choice& c) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, c.order);
  return {top, __reduce_min_sync(0xffffffffu, c.order == top ? c.column : INT32_MAX)};
}

// The raw logits of a unit are pairs of 16 bits, or fp32.

// -infinity where a bit of `keep` is not set.
template <int DT>
__device__ __forceinline__ void keep_only(uint32_t (&w)[4], uint32_t keep) {
  constexpr uint32_t LOWEST = DT == SPECTRA_DT_F32 ? 0xFF800000u : DT == SPECTRA_DT_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == SPECTRA_DT_F32) {
      w[i] = keep >> i & 1u ? w[i] : LOWEST;
    } else {
      const uint32_t two = keep >> (2 * i) & 3u, mask = ((two | two << 15) & 0x10001u) * 0xFFFFu;
      w[i] = (w[i] & mask) | (LOWEST & ~mask);
    }
  }
}
// The largest of both halves, a NaN where there is one.
template <int DT>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == SPECTRA_DT_BF16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (DT == SPECTRA_DT_F16)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT>
__device__ __forceinline__ float element(const uint32_t (&w)[4], int e) {
  if constexpr (DT == SPECTRA_DT_F32) return __uint_as_float(w[e]);
  return bits_to_float(w[e >> 1] >> (16 * (e & 1)) & 0xFFFFu, DT);
}
template <int DT>
__device__ __forceinline__ float top_of(const uint32_t (&w)[4]) {
  uint32_t t = max2<DT>(max2<DT>(w[0], w[1]), max2<DT>(w[2], w[3]));
  if constexpr (DT != SPECTRA_DT_F32) t = max2<DT>(t, t >> 16) & 0xFFFFu;
  return bits_to_float(t, DT);
}

// The cluster's barrier in two halves (arriving releases, waiting acquires).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

struct Penalties {
  float rep, freq, pres;
  const float* bias;
};
__device__ __forceinline__ float ruled(float x, uint32_t w, const Penalties& p) {
  const uint32_t times = w & kCountMask;
  if (w & (kPrompt | kCountMask)) x = x > 0.f ? __fdiv_rn(x, p.rep) : __fmul_rn(x, p.rep);
  if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.freq, float(times))), p.pres);
  if (w >> kSlot) x = __fadd_rn(x, p.bias[(w >> kSlot) - 1]);
  return x;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) logits_kernel(LogitArgs a) {
  namespace cg = cooperative_groups;
  constexpr int PER = kPer<DT>, ALL = (1 << PER) - 1, SIZE = DT == SPECTRA_DT_F32 ? 4 : 2;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t words[];  // [kChunk<DT>]
  uint16_t* met = reinterpret_cast<uint16_t*>(words + kChunk<DT>);  // [kChunk<DT>] words of the tokens met
  __shared__ int s_met;
  __shared__ Choice s_best[kWarps], s_rows_best[kMaxCluster];
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t m = blockIdx.y;
  const SpectraLogitRules& r = a.r;
  const uint8_t* row = static_cast<const uint8_t*>(a.x) + m * a.x_rs * SIZE;
  // unit u: columns u PER - shift ..: 16 bytes at a 16-byte address, the first at a multiple of a turn's 128 bytes,
  // so that no two CTAs write into one sector
  const int shift = int(reinterpret_cast<uintptr_t>(row) % (16 << kTurn)) / SIZE;
  const int N = int(a.N), offset = int(a.idx_offset);
  // local unit l of this CTA: unit ((l >> kTurn) * CTAs + rank) << kTurn | l % (1 << kTurn)
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank()), ctas_log2 = 31 - __clz(ctas);
  const int turns = (((N + shift + PER - 1) / PER) + (1 << kTurn) - 1) >> kTurn;
  const int mine = ((turns - rank + ctas - 1) >> ctas_log2) << kTurn;  // local units (a few past the row's end)
  auto first_column = [&](int l) {
    return (((((l >> kTurn) << ctas_log2) + rank) << kTurn) + (l & ((1 << kTurn) - 1))) * PER - shift;
  };
  uint8_t* out = static_cast<uint8_t*>(a.out) + m * a.out_rs * (a.out_dtype == SPECTRA_DT_F32 ? 4 : 2);
  const bool as_units = a.out_dtype == DT && int(reinterpret_cast<uintptr_t>(out) % 16) / SIZE == shift % PER;
  const int len = !r.ids ? 0 : (r.lengths ? clamp_len(r.lengths[m], r.max_ids) : int(r.max_ids));
  const int prompt = r.prompt_lengths ? clamp_len(r.prompt_lengths[m], len) : 0;
  const int* ids = r.ids + m * r.ids_stride;
  const int* allowed = r.allowed ? r.allowed + m * r.allowed_stride : nullptr;
  const int* bias_ids = r.bias_ids + m * r.bias_ids_stride;
  const Penalties pen = {r.repetition ? r.repetition[m] : 1.f, r.frequency ? r.frequency[m] : 0.f,
                         r.presence ? r.presence[m] : 0.f, r.bias + m * r.bias_stride};
  const bool counted = len > 0 || r.n_bias > 0;
  if (a.idx) cluster_arrive();  // (waited for before the first CTA's memory is written)
  auto may_follow = [&](int n) { return !allowed || (uint32_t(__ldcg(allowed + ((n + offset) >> 5))) >> ((n + offset) & 31) & 1u); };
  Choice best = {0, INT32_MAX};
  auto consider = [&](float v, int n) {
    const uint32_t o = order_of(v);
    if (o > best.order || (o == best.order && n < best.column)) best = {o, n};
  };
  for (int c0 = 0; c0 < mine; c0 += kThreads * kUnits) {
    const int c1 = min(mine, c0 + kThreads * kUnits), columns = (c1 - c0) * PER;
    const int column0 = first_column(c0 + tid), step = (kThreads * PER) << ctas_log2;
    uint32_t raw[kUnits][4], word0[kUnits], word1[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int l = c0 + tid + k * kThreads, n0 = column0 + k * step;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[k][i] = 0;
      word0[k] = word1[k] = ~0u;
      if (l < c1 && n0 >= 0 && n0 + PER <= N) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(row + int64_t(n0) * SIZE));
        raw[k][0] = v.x; raw[k][1] = v.y; raw[k][2] = v.z; raw[k][3] = v.w;
        if (allowed) {
          const int t = n0 + offset;
          word0[k] = uint32_t(__ldcg(allowed + (t >> 5)));
          if ((t & 31) > 32 - PER) word1[k] = uint32_t(__ldcg(allowed + (t >> 5) + 1));
        }
      } else if (l < c1) {  // cut at an end of the row: one by one, columns outside as if they were not allowed
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int n = n0 + e;
          if (n < 0 || n >= N) continue;
          raw[k][DT == SPECTRA_DT_F32 ? e : e >> 1] |= load_bits_cg(row, n, DT) << (DT == SPECTRA_DT_F32 ? 0 : 16 * (e & 1));
          bits |= uint32_t(may_follow(n)) << e;
        }
        const int at = (n0 + offset) & 31;
        word0[k] = bits << at;
        word1[k] = at > 32 - PER ? bits >> (32 - at) : 0;
      }
    }
    // the first ids, before the row's length is known (a row of ids is max_ids long)
    int early[kFlight], early_bias = -1;
#pragma unroll
    for (int k = 0; k < kFlight; ++k) early[k] = tid + k * kThreads < r.max_ids ? __ldcg(ids + tid + k * kThreads) : -1;
    if (tid < r.n_bias) early_bias = __ldcg(bias_ids + tid);
    uint32_t own = 0;  // which of the thread's columns were met
    if (counted) {
      for (int i = tid; i < columns / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) s_met = 0;
      // a token's word, or -1: not of this CTA and chunk
      auto word_of = [&](int id) {
        const unsigned n = unsigned(id - offset), at = n + shift, turn = at / (PER << kTurn);  // (a negative id is past N)
        const unsigned w = (turn >> ctas_log2) * (PER << kTurn) + at % (PER << kTurn) - c0 * PER;
        return n < unsigned(N) && (turn & unsigned(ctas - 1)) == unsigned(rank) && w < unsigned(columns) ? int(w) : -1;
      };
      __syncthreads();
      for (int i0 = tid; i0 < len; i0 += kFlight * kThreads) {
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          const int w = i0 + k * kThreads < len ? word_of(early[k]) : -1;
          if (w < 0) continue;
          if (i0 + k * kThreads < prompt)
            atomicOr(words + w, kPrompt);
          else
            atomicAdd(words + w, 1u);
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          const int i = i0 + (kFlight + k) * kThreads;
          if (i < len) early[k] = __ldcg(ids + i);
        }
      }
      __syncthreads();
      if (r.n_bias > 0) {
        for (int i = tid; i < r.n_bias; i += kThreads) {
          const int w = word_of(i == tid ? early_bias : __ldcg(bias_ids + i));
          if (w < 0) continue;
          // (the low bits are settled, so the larger word is the later entry)
          atomicMax(words + w, (words[w] & kLow) | uint32_t(i + 1) << kSlot);
        }
        __syncthreads();
      }
      // the tokens met, side by side
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int w = (tid + k * kThreads) * PER;
        if (w < columns) {
#pragma unroll
          for (int e = 0; e < PER; e += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(words + w + e);
            own |= uint32_t(min(v.x, 1u) | min(v.y, 1u) << 1 | min(v.z, 1u) << 2 | min(v.w, 1u) << 3) << (k * PER + e);
          }
        }
      }
      int before = __popc(own);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      int base = 0;
      if (lane == 31 && before) base = atomicAdd(&s_met, before);
      int slot = __shfl_sync(0xffffffffu, base, 31) + before - __popc(own);
      for (uint32_t left = own; left; left &= left - 1) {
        const int i = __ffs(left) - 1;
        met[slot++] = uint16_t((tid + i / PER * kThreads) * PER + i % PER);
      }
      __syncthreads();
      for (int i = tid; i < s_met; i += kThreads) {
        const int w = met[i], n = first_column(c0 + w / PER) + w % PER;
        words[w] = __float_as_uint(ruled(load_as_float_cg(row, n, DT), words[w], pen));
      }
      __syncthreads();  // (the row is written from here on, and may be the logits themselves)
    }
    float top = -INFINITY;  // of the thread's units, the first that has it, and what it keeps
    uint32_t top_keep = 0, top_raw[4] = {0, 0, 0, 0};
    int top_column = 0;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int n0 = column0 + k * step;
      if (c0 + tid + k * kThreads >= c1) break;
      const uint32_t keep = __funnelshift_r(word0[k], word1[k], (n0 + offset) & 31) & ~(own >> (k * PER)) & ALL;
      if (keep != ALL) keep_only<DT>(raw[k], keep);
      if (a.out) {
        if (as_units && n0 >= 0 && n0 + PER <= N) {
          *reinterpret_cast<uint4*>(out + int64_t(n0) * SIZE) = make_uint4(raw[k][0], raw[k][1], raw[k][2], raw[k][3]);
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (n0 + e >= 0 && n0 + e < N) store_from_float(out, n0 + e, a.out_dtype, element<DT>(raw[k], e));
        }
      }
      const float t = top_of<DT>(raw[k]);
      if (keep && (!top_keep || t > top || (t != t && top == top))) {
        top = t;
        top_keep = keep;
        top_column = n0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top_raw[i] = raw[k][i];
      }
    }
    if (a.idx && top_keep) {
      // the first column that has it (where that is -infinity, among the kept)
      int at = __ffs(top_keep) - 1;
      if (top > -INFINITY) {
#pragma unroll
        for (int e = PER - 1; e >= 0; --e) at = element<DT>(top_raw, e) == top ? e : at;
      } else if (top != top) {
#pragma unroll
        for (int e = PER - 1; e >= 0; --e) at = element<DT>(top_raw, e) != element<DT>(top_raw, e) ? e : at;
      }
      consider(top, top_column + at);
    }
    if (counted) {
      __syncthreads();
      for (int i = tid; i < s_met; i += kThreads) {
        const int w = met[i], n = first_column(c0 + w / PER) + w % PER;
        const bool ok = may_follow(n);
        const float y = ok ? __uint_as_float(words[w]) : -INFINITY;
        if (a.out) store_from_float(out, n, a.out_dtype, y);
        if (ok) consider(y, n);
      }
      __syncthreads();  // before the next chunk clears the words
    }
  }
  if (!a.idx) return;  // (the same for every CTA)
  best = best_of_warp(best);
  if (lane == 0) s_best[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = lane < kWarps ? s_best[lane] : Choice{0, INT32_MAX};
    best = best_of_warp(best);
  }
  cluster_wait();  // every CTA of the cluster runs
  if (tid == 0) *cluster.map_shared_rank(&s_rows_best[rank], 0) = best;
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && warp == 0) {
    best = best_of_warp(lane < ctas ? s_rows_best[lane] : Choice{0, INT32_MAX});
    if (lane == 0) {
      a.idx[m] = best.order ? best.column + a.idx_offset : -1;
      if (a.val) a.val[m] = value_of(best.order);
    }
  }
}

// ------------------------------------------------------------ many rows
constexpr int kSliceUnits = kThreads * kUnits;         // of a slice
constexpr int kMaxTableLog2 = 13;                      // slots of a row's table
constexpr int64_t kMaxListed = (1 << kMaxTableLog2) * 2 / 3;  // ids and biases of a row
constexpr int64_t kMaxMet = (1 << 18) + 4096;          // columns of a row, a bit each
constexpr uint32_t kFree = ~0u;
constexpr int kMostThreads = 1024;                     // of a row's CTA

// A thread's unit at column n0: its logits and which of them may follow (columns outside the row may not).
template <int DT>
__device__ __forceinline__ uint32_t load_unit(const uint8_t* row, const int* allowed, int n0, int N, int offset, uint32_t (&raw)[4]) {
  constexpr int PER = kPer<DT>, ALL = (1 << PER) - 1, SIZE = DT == SPECTRA_DT_F32 ? 4 : 2;
  raw[0] = raw[1] = raw[2] = raw[3] = 0;
  if (n0 >= 0 && n0 + PER <= N) {
    const uint4 v = __ldcg(reinterpret_cast<const uint4*>(row + int64_t(n0) * SIZE));
    raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
    if (!allowed) return ALL;
    const int t = n0 + offset;
    const uint32_t w0 = uint32_t(__ldcg(allowed + (t >> 5)));
    const uint32_t w1 = (t & 31) > 32 - PER ? uint32_t(__ldcg(allowed + (t >> 5) + 1)) : 0;
    return __funnelshift_r(w0, w1, t & 31) & ALL;
  }
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int n = n0 + e;
    if (n < 0 || n >= N) continue;
    raw[DT == SPECTRA_DT_F32 ? e : e >> 1] |= load_bits_cg(row, n, DT) << (DT == SPECTRA_DT_F32 ? 0 : 16 * (e & 1));
    bits |= (allowed ? uint32_t(__ldcg(allowed + ((n + offset) >> 5))) >> ((n + offset) & 31) & 1u : 1u) << e;
  }
  return bits;
}

// The first column that has `top`, the largest of a unit's kept columns (the others are -infinity).
template <int DT>
__device__ __forceinline__ int first_of(const uint32_t (&raw)[4], uint32_t keep, float top) {
  int at = __ffs(keep) - 1;
  if (top > -INFINITY) {
#pragma unroll
    for (int e = kPer<DT> - 1; e >= 0; --e) at = element<DT>(raw, e) == top ? e : at;
  } else if (top != top) {
#pragma unroll
    for (int e = kPer<DT> - 1; e >= 0; --e) at = element<DT>(raw, e) != element<DT>(raw, e) ? e : at;
  }
  return at;
}

__device__ __forceinline__ bool before(const Choice& a, const Choice& b) {
  return a.order > b.order || (a.order == b.order && a.column < b.column);
}

// The best of the CTA's threads, in its first warp.
__device__ __forceinline__ Choice best_of_cta(Choice c, Choice* s_best) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  c = best_of_warp(c);
  if (lane == 0) s_best[warp] = c;
  __syncthreads();
  if (warp == 0) c = best_of_warp(lane < int(blockDim.x >> 5) ? s_best[lane] : Choice{0, INT32_MAX});
  return c;
}

// Column of unit u of a row is u PER - shift: the first unit starts at a multiple of 128 bytes.
template <int DT>
__device__ __forceinline__ int row_shift(const uint8_t* row) {
  return int(reinterpret_cast<uintptr_t>(row) % 128) / (DT == SPECTRA_DT_F32 ? 4 : 2);
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 3) rows_kernel(LogitArgs a) {
  constexpr int PER = kPer<DT>, ALL = (1 << PER) - 1, SIZE = DT == SPECTRA_DT_F32 ? 4 : 2;
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const int64_t m = blockIdx.y;
  const uint8_t* row = static_cast<const uint8_t*>(a.x) + m * a.x_rs * SIZE;
  uint8_t* out = static_cast<uint8_t*>(a.out) + m * a.out_rs * (a.out_dtype == SPECTRA_DT_F32 ? 4 : 2);
  const int* allowed = a.r.allowed ? a.r.allowed + m * a.r.allowed_stride : nullptr;
  const int N = int(a.N), offset = int(a.idx_offset), shift = row_shift<DT>(row);
  const bool as_units = a.out_dtype == DT && int(reinterpret_cast<uintptr_t>(out) % 16) / SIZE == shift % PER;
  const int column0 = (int(blockIdx.x) * kSliceUnits + int(threadIdx.x)) * PER - shift;
  uint32_t raw[kUnits][4], keep[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k)
    keep[k] = column0 + k * kThreads * PER < N ? load_unit<DT>(row, allowed, column0 + k * kThreads * PER, N, offset, raw[k]) : 0;
  Choice best = {0, INT32_MAX};
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int n0 = column0 + k * kThreads * PER;
    if (n0 >= N) break;
    if (keep[k] != ALL) keep_only<DT>(raw[k], keep[k]);
    if (a.out) {
      if (as_units && n0 >= 0 && n0 + PER <= N) {
        *reinterpret_cast<uint4*>(out + int64_t(n0) * SIZE) = make_uint4(raw[k][0], raw[k][1], raw[k][2], raw[k][3]);
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (n0 + e >= 0 && n0 + e < N) store_from_float(out, n0 + e, a.out_dtype, element<DT>(raw[k], e));
      }
    }
    if (a.idx && keep[k]) {
      const float top = top_of<DT>(raw[k]);
      const Choice c = {order_of(top), n0 + PER};  // (its place is looked for below, if this is the best)
      if (c.order > best.order) best = c;
    }
  }
  if (!a.idx) return;
  // the highest, and where it is found the first column that has it
  const uint32_t top = __reduce_max_sync(0xffffffffu, best.order);
  if (best.order != top) best = {0, INT32_MAX};
  if (best.order) {
#pragma unroll
    for (int k = kUnits - 1; k >= 0; --k) {
      if (!keep[k]) continue;
      const float t = top_of<DT>(raw[k]);
      if (order_of(t) == best.order) best.column = column0 + k * kThreads * PER + first_of<DT>(raw[k], keep[k], t);
    }
  }
  best = best_of_warp(best);
  if (threadIdx.x % 32 == 0) a.tops[(m * gridDim.x + blockIdx.x) * kWarps + threadIdx.x / 32] = make_uint2(best.order, uint32_t(best.column));
}

template <int DT>
__global__ void __launch_bounds__(kMostThreads) rules_kernel(LogitArgs a, int parts, int slots_log2) {
  constexpr int PER = kPer<DT>, SIZE = DT == SPECTRA_DT_F32 ? 4 : 2;
  extern __shared__ __align__(16) uint32_t keys[];  // [slots] columns, kFree; their words; a bit per column; the slots taken
  __shared__ Choice s_best[kMostThreads / 32], s_rows_best[kMaxCluster];
  __shared__ int s_parts[(kMaxMet / (kSliceUnits * 4) + 2) * kWarps], s_again, s_taken;
  const int slots = 1 << slots_log2, tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
  uint32_t *words = keys + slots, *met = words + slots;
  uint16_t* taken = reinterpret_cast<uint16_t*>(met + int(a.N) / 32 + 2);
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());  // of the row: each has every ctas-th column
  const int64_t m = blockIdx.y;
  const SpectraLogitRules& r = a.r;
  const int N = int(a.N), offset = int(a.idx_offset), met_words = N / 32 + 2;
  const bool counted = slots_log2 > 0;
  Choice best = {0, INT32_MAX};
  auto consider = [&](float v, int n) {
    const Choice c = {order_of(v), n};
    if (before(c, best)) best = c;
  };
  // The lists come from kernels before the one that passes over the rows, which started after them: this part
  // need not wait for it.
  const int len = !r.ids ? 0 : (r.lengths ? clamp_len(__ldcg(r.lengths + m), r.max_ids) : int(r.max_ids));
  const int prompt = r.prompt_lengths ? clamp_len(__ldcg(r.prompt_lengths + m), len) : 0;
  const int *ids = r.ids + m * r.ids_stride, *bias_ids = r.bias_ids + m * r.bias_ids_stride;
  const Penalties pen = {r.repetition ? __ldcg(r.repetition + m) : 1.f, r.frequency ? __ldcg(r.frequency + m) : 0.f,
                         r.presence ? __ldcg(r.presence + m) : 0.f, r.bias + m * r.bias_stride};
  if (tid == 0) s_again = s_taken = 0;
  if (counted) {
    for (int i = tid; i < slots / 4; i += threads) {
      reinterpret_cast<uint4*>(keys)[i] = make_uint4(kFree, kFree, kFree, kFree);
      reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    }
    for (int i = tid; i < met_words; i += threads) met[i] = 0;
    // a token's slot, which it takes if it is the first; -1: none of these columns.  (A third of the slots stay free.)
    auto slot_of = [&](int id) {
      const unsigned n = unsigned(id - offset);  // (a negative id is past N)
      if (n >= unsigned(N) || (n & unsigned(ctas - 1)) != unsigned(rank)) return -1;
      unsigned slot = n * 0x9E3779B1u >> (32 - slots_log2);
      for (;; slot = (slot + 1) & unsigned(slots - 1)) {
        uint32_t key = *static_cast<volatile uint32_t*>(keys + slot);
        if (key == kFree) {
          key = atomicCAS(keys + slot, kFree, n);
          if (key == kFree) {  // taken: the lanes that take one now have places side by side in the list
            const cg::coalesced_group now = cg::coalesced_threads();
            int at = 0;
            if (now.thread_rank() == 0) at = atomicAdd(&s_taken, int(now.size()));
            taken[now.shfl(at, 0) + now.thread_rank()] = uint16_t(slot);
            return int(slot);
          }
        }
        if (key == n) return int(slot);
      }
    };
    __syncthreads();
    for (int i0 = tid; i0 < len; i0 += kFlight * threads) {
      int id[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) id[k] = i0 + k * threads < len ? __ldcg(ids + i0 + k * threads) : -1;
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int slot = id[k] < 0 ? -1 : slot_of(id[k]);
        if (slot < 0) continue;
        if (i0 + k * threads < prompt)
          atomicOr(words + slot, kPrompt);
        else
          atomicAdd(words + slot, 1u);
      }
    }
    __syncthreads();
    for (int i = tid; i < r.n_bias; i += threads) {
      const int id = __ldcg(bias_ids + i), slot = id < 0 ? -1 : slot_of(id);
      // (the low bits are settled, so the larger word is the later entry)
      if (slot >= 0) atomicMax(words + slot, (words[slot] & kLow) | uint32_t(i + 1) << kSlot);
    }
    __syncthreads();
  }
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const uint8_t* row = static_cast<const uint8_t*>(a.x) + m * a.x_rs * SIZE;
  uint8_t* out = static_cast<uint8_t*>(a.out) + m * a.out_rs * (a.out_dtype == SPECTRA_DT_F32 ? 4 : 2);
  const int* allowed = r.allowed ? r.allowed + m * r.allowed_stride : nullptr;
  if (counted) {
    for (int j0 = tid; j0 < s_taken; j0 += kFlight * threads) {
      uint32_t n[kFlight], bits[kFlight], word[kFlight];
      int slot[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        slot[k] = j0 + k * threads < s_taken ? taken[j0 + k * threads] : -1;
        n[k] = bits[k] = 0;
        word[k] = ~0u;
        if (slot[k] < 0) continue;
        n[k] = keys[slot[k]];
        bits[k] = load_bits_cg(row, n[k], DT);
        if (allowed) word[k] = uint32_t(__ldcg(allowed + ((n[k] + offset) >> 5)));
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        if (slot[k] < 0) continue;
        atomicOr(met + (n[k] >> 5), 1u << (n[k] & 31));
        const bool ok = word[k] >> ((n[k] + offset) & 31) & 1u;
        const float y = ok ? ruled(bits_to_float(bits[k], DT), words[slot[k]], pen) : -INFINITY;
        if (a.out) store_from_float(out, n[k], a.out_dtype, y);
        if (ok) consider(y, int(n[k]));
      }
    }
  }
  if (!a.idx) return;
  if (ctas > 1) cluster.sync(); else __syncthreads();
  // ---- the parts' maxima, each CTA some of them; those of tokens met are looked for again, by a warp each
  auto met_at = [&](int i) {
    uint32_t bits = 0;
    for (int c = 0; c < ctas; ++c) bits |= ctas > 1 ? *cluster.map_shared_rank(met + i, c) : met[i];
    return bits;
  };
  for (int i = rank + tid * ctas; i < parts; i += threads * ctas) {
    const uint2 top = __ldcg(a.tops + m * parts + i);
    const Choice c = {top.x, int(top.y)};
    if (!c.order) continue;
    if (counted && (met_at(c.column >> 5) >> (c.column & 31) & 1u))
      s_parts[atomicAdd(&s_again, 1)] = i;
    else if (before(c, best))
      best = c;
  }
  __syncthreads();
  const int shift = row_shift<DT>(row);
  for (int j = tid >> 5; j < s_again; j += threads >> 5) {
    const int slice = s_parts[j] / kWarps, column0 = (slice * kSliceUnits + s_parts[j] % kWarps * 32 + lane) * PER - shift;
    uint32_t raw[kUnits][4], keep[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      keep[k] = column0 + k * kThreads * PER < N ? load_unit<DT>(row, allowed, column0 + k * kThreads * PER, N, offset, raw[k]) : 0;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (!keep[k]) continue;
      const int n0 = column0 + k * kThreads * PER;
      const int first = max(n0, 0) >> 5, bit = n0 - first * 32;  // (a unit that begins before the row: bit < 0)
      const uint32_t m0 = met_at(first), m1 = bit > 32 - PER ? met_at(first + 1) : 0;
      keep[k] &= ~(bit >= 0 ? __funnelshift_r(m0, m1, bit) : m0 << -bit);
      if (!keep[k]) continue;
      keep_only<DT>(raw[k], keep[k]);
      const float top = top_of<DT>(raw[k]);
      if (order_of(top) >= best.order) consider(top, n0 + first_of<DT>(raw[k], keep[k], top));
    }
  }
  best = best_of_cta(best, s_best);
  if (ctas > 1) {
    if (tid == 0) *cluster.map_shared_rank(&s_rows_best[rank], 0) = best;
    cluster.sync();
    if (rank == 0 && tid < 32) best = best_of_warp(lane < ctas ? s_rows_best[lane] : Choice{0, INT32_MAX});
  }
  if (rank == 0 && tid == 0) {
    a.idx[m] = best.order ? best.column + a.idx_offset : -1;
    if (a.val) a.val[m] = value_of(best.order);
  }
}

// CTAs per row of the one kernel: as few as hold the row at once.
int ctas_of(int64_t N, int dt) {
  const int64_t chunk = int64_t(kThreads) * kUnits * (dt == SPECTRA_DT_F32 ? 4 : 8);
  int ctas = 1;
  while (ctas < kMaxCluster && ctas * chunk < N) ctas *= 2;
  return ctas;
}

template <int DT>
int launch_few(const LogitArgs& a, cudaStream_t st) {
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  const int smem = kChunk<DT> * 6;
  e = once.run(dev, [&] { return cudaFuncSetAttribute(logits_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (e != cudaSuccess) return cuda_status(e);
  // (each CTA reads the lists; more of them while there are SMs without one)
  int ctas = ctas_of(a.N, DT);
  while (ctas < kMaxCluster && a.M * ctas < device_sms(dev)) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas), unsigned(a.M));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, logits_kernel<DT>, a));
}

bool has_lists(const SpectraLogitRules& r) { return r.max_ids > 0 || r.n_bias > 0; }

// One kernel for all while the GPU holds its CTAs at once (kAtOnce of them on a B200).  Measured, lists of 5000 ids and
// 300 biases, 128256 columns: 32 rows 14.5 us with one kernel, 20.9 with two; 64 rows 26.8 and 26.1; 128 rows 48.9
// and 39.8.  Masks alone, 64 rows: 10.5 and 8.6.  32000 columns, 128 rows: 16.8 and 29.3.  The lists' width decides, as
// what they hold is known on the device alone: 333 rows of 50001 with 200 ids each take 19.7 us in lists 200 wide, 28.0
// in ones of 5461, 43.7 in wider ones, by the one kernel.
constexpr int64_t kAtOnce = 296;
bool many_rows(const SpectraLogitRules& r, int64_t M, int64_t N, int dt) {
  return M * ctas_of(N, dt) > kAtOnce && r.max_ids + r.n_bias <= kMaxListed && N <= kMaxMet - 64;
}
int64_t slices_of(int64_t N, int dt) {
  const int64_t columns = int64_t(kSliceUnits) * (dt == SPECTRA_DT_F32 ? 4 : 8), shift = dt == SPECTRA_DT_F32 ? 31 : 63;
  return (N + shift + columns - 1) / columns;
}

template <int DT>
int launch_many(const LogitArgs& a, cudaStream_t st) {
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  constexpr int kMost = (10 << kMaxTableLog2) + int(kMaxMet / 8) + 8;
  e = once.run(dev, [&] { return cudaFuncSetAttribute(rules_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost); });
  if (e != cudaSuccess) return cuda_status(e);
  const int slices = int(slices_of(a.N, DT));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(slices), unsigned(a.M));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, rows_kernel<DT>, a);
  if (e != cudaSuccess || (!has_lists(a.r) && !a.idx)) return cuda_status(e);
  int log2 = 0;
  size_t smem = 0;
  if (has_lists(a.r)) {
    for (log2 = 6; (int64_t(2) << log2) < 3 * (a.r.max_ids + a.r.n_bias); ++log2) {}
    smem = (size_t(10) << log2) + (size_t(a.N) / 32 + 2) * 4;
  }
  // As many CTAs per row as leave none of the SMs idle, where the lists are long enough to share.  Measured, 40 rows of
  // 128256: 100 ids 10.4 us (11.7 with lists shared from 128 slots a CTA on), 300 ids 12.7 (21.5 from 2048 on), 600 ids
  // 14.4 (20.4 from 2048 on).
  int ctas = 1;
  while (ctas < kMaxCluster && a.M * ctas * 2 <= device_sms(dev) && (1 << log2) >= 512 * ctas) ctas *= 2;
  cfg.gridDim = dim3(unsigned(ctas), unsigned(a.M));
  cfg.blockDim = dim3(unsigned(std::min(kMostThreads, std::max(256, (1 << log2) / 8))));  // 8 slots a thread
  cfg.dynamicSmemBytes = smem;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, rules_kernel<DT>, a, slices * kWarps, log2));
}

}  // namespace

size_t logits_workspace_bytes(const SpectraLogitRules& r, int64_t M, int64_t N, int x_dtype, bool tokens) {
  return tokens && many_rows(r, M, N, x_dtype) ? size_t(M) * slices_of(N, x_dtype) * kWarps * sizeof(uint2) : 0;
}

int launch_logits(const LogitArgs& a, cudaStream_t st) {
  if (a.M == 0) return SPECTRA_OK;
  const bool many = many_rows(a.r, a.M, a.N, a.x_dtype);
  if (a.x_dtype == SPECTRA_DT_BF16) return many ? launch_many<SPECTRA_DT_BF16>(a, st) : launch_few<SPECTRA_DT_BF16>(a, st);
  if (a.x_dtype == SPECTRA_DT_F16) return many ? launch_many<SPECTRA_DT_F16>(a, st) : launch_few<SPECTRA_DT_F16>(a, st);
  return many ? launch_many<SPECTRA_DT_F32>(a, st) : launch_few<SPECTRA_DT_F32>(a, st);
}

}  // namespace spectra
