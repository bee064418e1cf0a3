// Block index of the paged INT4 KV cache, and the choice of blocks by it, for
// sm_100a.
//
// Index, of each block of block_size tokens and each head:
//   hi_d = max k_d, lo_d = min k_d over the block's keys k = (q - z) s
//   S = least 2^e with max(|hi|, |lo|) <= 127 S;  H = ceil(hi / S), L = floor(lo / S)
// A largest value does not depend on the order it is looked for in, (q - z) s has 15
// bits and S is a power of two: nothing is rounded before the two outward roundings.
//
// Choice, for a token and a key/value head whose query heads have codes c_h:
//   score(j) = S_j max_h sum_d (c_hd > 0 ? c_hd H_jd : c_hd L_jd)
// an upper bound of c_h . k for every key of the block and every head.  (Each head's
// codes have a step of its own, which is left out: a ranking, no bound of q . k.)  The sum is
// max(c, 0) . H + min(c, 0) . L, a product of integers below 2^22, so scores are
// exact in fp32 and the choice does not depend on the order of the sums.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "copy_ring.h"
#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

__device__ int g_paged_index_timeouts = 0;

namespace {

// 2^e, the least with most <= 127 * 2^e, e >= -126; 1 for 0 (most: not negative, finite).
__device__ __forceinline__ float range_step(float most) {
  const uint32_t bits = __float_as_uint(most);
  if (bits == 0) return 1.f;
  // 127 = 1.984375 * 2^6, with mantissa 0x7E0000
  const int e = int(bits >> 23) - 6 + ((bits & 0x7FFFFFu) > 0x7E0000u);
  return __uint_as_float(uint32_t(max(e, 1)) << 23);
}
// 1 / 2^e exactly, for e in [-126, 126]
__device__ __forceinline__ float inverse_step(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// ------------------------------------------------------------ index
// A warp has one block of one head.  A lane has one word of codes, 8 features, of every
// ROWS-th token, so that little is left to put together.  A nibble under an exponent is
// 2048 + q where it lies in bits 12-15 and 128 + q in bits 16-19, so one fma with
// -(2048 + z) s or -(128 + z) s makes it (q - z) s: 23 and 19 bits, exact.
//
// Bound by instructions, about 40 for a word of two tokens (issue slots 64 % taken, ALU 57 %).
// Measured: 6 ragged prompts up to 16384, 8 heads of 128, blocks of 64: 20.3 us with the cache
// in HBM (1.7 TB/s; loads straight from memory 25.7), one token of 128 sequences 3.9 us.
constexpr int kIndexWarps = 4;  // of a CTA

// 2048 + q of bits 12-15, 128 + q of bits 16-19 (the exponents in registers: mask-and-or is one instruction then).
__device__ __forceinline__ float nibble_at_12(uint32_t w, uint32_t exponent) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x0000F000, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(exponent));
  return __uint_as_float(r);
}
__device__ __forceinline__ float nibble_at_16(uint32_t w, uint32_t exponent) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F0000, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(exponent));
  return __uint_as_float(r);
}
__device__ __forceinline__ uint32_t in_register(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The range of a word's features over the tokens that a lane has seen.
struct Range {
  float hi[8], lo[8], finite;  // finite: 0, or NaN once a scale was not
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      hi[i] = -INFINITY;
      lo[i] = INFINITY;
    }
    finite = 0.f;
  }
  // two tokens: words, scales, zero points
  __device__ __forceinline__ void add(const uint32_t (&w)[2], const float (&scale)[2], const float (&zero)[2], uint32_t e12, uint32_t e16) {
    float v[2][8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float s = scale[x], c12 = -(2048.f + zero[x]) * s, c16 = -(128.f + zero[x]) * s;
      finite = fmaf(s, 0.f, finite);
      const uint32_t q[4] = {w[x] << 12, w[x] << 4, w[x] >> 4, w[x] >> 12};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[x][2 * i] = fmaf(nibble_at_12(q[i], e12), s, c12);
        v[x][2 * i + 1] = fmaf(nibble_at_16(q[i], e16), s, c16);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      hi[i] = max3(hi[i], v[0][i], v[1][i]);
      lo[i] = min3(lo[i], v[0][i], v[1][i]);
    }
  }
};

// A lane's word of a token and which of the tokens it takes.
template <int G>
struct LaneWord {
  static constexpr int W = 4 * G, ROWS = G == 8 ? 1 : G >= 3 ? 2 : 8 / G;  // words of a token, tokens of a warp at once
  int row, word, g;
  __device__ __forceinline__ explicit LaneWord(int lane) {
    row = min(lane / W, ROWS - 1);
    word = lane < ROWS * W ? lane % W : 0;
    g = word % G;
  }
  // lanes of the same word become one: lane word has it
  __device__ __forceinline__ void join_rows(Range& r) const {
#pragma unroll
    for (int o = W; o < ROWS * W; o *= 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r.hi[i] = fmaxf(r.hi[i], __shfl_down_sync(0xffffffffu, r.hi[i], o));
        r.lo[i] = fminf(r.lo[i], __shfl_down_sync(0xffffffffu, r.lo[i], o));
      }
    }
  }
  // the index of a block, from the lanes that have a word's whole range
  __device__ __forceinline__ void store(const PagedIndexArgs& a, int64_t slot, const Range& r, bool bad, int lane) const {
    constexpr int D = 32 * G;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fabsf(r.hi[i]), fabsf(r.lo[i])));
    // (magnitudes, as whole numbers in the order of the values)
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < W && !bad ? __float_as_uint(top) : 0u));
    const float step = range_step(top), inv = inverse_step(step);
    if (lane < W) {
      uint32_t up[2] = {0, 0}, down[2] = {0, 0};
      if (!bad) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          up[i >> 2] |= (uint32_t(int(ceilf(r.hi[i] * inv))) & 255u) << (8 * (i & 3));
          down[i >> 2] |= (uint32_t(int(floorf(r.lo[i] * inv))) & 255u) << (8 * (i & 3));
        }
      }
      const int d0 = g * 32 + word / G * 8;
      *reinterpret_cast<uint2*>(a.codes + slot * 2 * D + d0) = make_uint2(up[0], up[1]);
      *reinterpret_cast<uint2*>(a.codes + slot * 2 * D + D + d0) = make_uint2(down[0], down[1]);
    }
    if (lane == 0) a.scales[slot] = bad ? INFINITY : step;
  }
};

// The blocks of sequence b that its new tokens filled: j0 .. end - 1 (end >= j0, also where the sequence goes on
// past the bound: the counts are added up).
__device__ __forceinline__ void filled_blocks(const PagedIndexArgs& a, int b, int& j0, int& end) {
  int64_t first;
  int count;
  new_tokens(a.c, b, first, count);
  const int held = a.c.seq_lens[b], len = min(held, a.c.limit);
  j0 = max(held - count, 0) >> a.block_log2;
  end = len > 0 && count > 0 ? max(len >> a.block_log2, j0) : j0;
}

// Few blocks: the four warps of a CTA share one, a quarter of its tokens each, straight from memory.
template <int G>
__global__ void __launch_bounds__(32 * kIndexWarps) paged_index_few_kernel(PagedIndexArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  using Word = LaneWord<G>;
  constexpr int W = Word::W, ROWS = Word::ROWS, FLIGHT = 8 / ROWS;  // 8 tokens of a warp are in flight: half a tile
  constexpr TileLayout L{G};
  __shared__ float2 s_part[kIndexWarps][8][W];  // [warp][feature of a word][word]: largest, smallest
  const PagedView& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Word at(lane);
  const uint32_t e12 = in_register(0x45000000u), e16 = in_register(0x43000000u);
  const int pl = c.page_log2 - a.block_log2, per_page = 1 << pl, tiles = 1 << (a.block_log2 - 4);
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    int j0, end;
    filled_blocks(a, b, j0, end);
    for (int64_t item = blockIdx.x; item < int64_t(end - j0) * c.kv_heads; item += gridDim.x) {
      const int j = j0 + int(item / c.kv_heads), h = int(item % c.kv_heads);
      const int page = c.tables[b * c.table_stride + (j >> pl)];
      if (unsigned(page) >= unsigned(c.num_pages)) continue;
      const int part = j & (per_page - 1);
      const uint8_t* t = c.pool + page * c.page_stride + ((int64_t(h) << (c.page_log2 - 4)) + int64_t(part) * tiles) * L.bytes();
      Range r;
      r.clear();
      const int share = tiles * 16 / kIndexWarps;
      for (int k0 = warp * share; k0 < (warp + 1) * share; k0 += 8) {
        const uint8_t* tile = t + (k0 >> 4) * L.bytes();
        const int half = k0 >> 3 & 1;
        uint32_t w[FLIGHT];
        float s[FLIGHT], z[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
          const int tok = k * ROWS + at.row;
          w[k] = __ldcg(reinterpret_cast<const uint32_t*>(tile + L.k_codes() + half * L.block()) + tok * W + at.word);
          s[k] = __half2float(__ldcg(reinterpret_cast<const __half*>(tile + L.k_scales()) + (8 * half + tok) * G + at.g));
          z[k] = float(__ldcg(tile + L.k_zeros() + (8 * half + tok) * G + at.g));
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; k += 2) {
          const int k1 = min(k + 1, FLIGHT - 1);  // (a flight of one token: the same again)
          r.add({w[k], w[k1]}, {s[k], s[k1]}, {z[k], z[k1]}, e12, e16);
        }
      }
      at.join_rows(r);
      bool bad = __any_sync(0xffffffffu, !(r.finite == 0.f));
      if (lane < W) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s_part[warp][i][lane] = make_float2(r.hi[i], r.lo[i]);
      }
      bad = __syncthreads_or(bad);
      if (warp == 0) {
        if (lane < W) {
#pragma unroll
          for (int x = 1; x < kIndexWarps; ++x)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              r.hi[i] = fmaxf(r.hi[i], s_part[x][i][lane].x);
              r.lo[i] = fminf(r.lo[i], s_part[x][i][lane].y);
            }
        }
        at.store(a, (int64_t(page) * c.kv_heads + h) * per_page + part, r, bad, lane);
      }
      __syncthreads();  // before the next block's are written
    }
  }
}

// Many blocks: a warp each, in pieces of 32 tokens that bulk copies bring into shared memory, the next piece
// while one is looked at.  Of a tile the key codes, and what lies from the key scales to the key zero points.
template <int G>
struct Piece {
  static constexpr int kTiles = 2, kCodes = 256 * G, kRest = 80 * G, kTile = kCodes + kRest, kBytes = kTiles * kTile;
  static constexpr int kStages = 3;
  static constexpr int kSmem = kIndexWarps * kStages * (kBytes + 8);
  static constexpr int kCtas = 224 * 1024 / (kSmem + 1024) < 8 ? 224 * 1024 / (kSmem + 1024) : 8;  // per SM
};

template <int G>
__global__ void __launch_bounds__(32 * kIndexWarps) paged_index_kernel(PagedIndexArgs a) {
  using Word = LaneWord<G>;
  using P = Piece<G>;
  constexpr int W = Word::W, ROWS = Word::ROWS;
  constexpr TileLayout L{G};
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ volatile int s_never;  // 0: each warp waits for its own copies
  constexpr int kSeqs = 32 * kIndexWarps;
  __shared__ int s_from[kSeqs], s_first[kSeqs], s_sum[kIndexWarps];
  const PagedView& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* stages = smem + warp * P::kStages * P::kBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kIndexWarps * P::kStages * P::kBytes) + warp * P::kStages;
  if (lane < P::kStages) sm100::mbar_init(bars + lane, 1);
  if (threadIdx.x == 0) s_never = 0;
  sm100::fence_mbar_init();
  __syncthreads();
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const Word at(lane);
  const uint32_t e12 = in_register(0x45000000u), e16 = in_register(0x43000000u);
  const int pl = c.page_log2 - a.block_log2, per_page = 1 << pl;
  const int pieces_log2 = a.block_log2 - 5;
  const int h = blockIdx.y, block0 = int(blockIdx.x) * kIndexWarps + warp, stride = int(gridDim.x) * kIndexWarps;
  CopyRing<P::kStages> ring;
  for (int b0 = 0; b0 < c.batch; b0 += kSeqs) {
    // ---- the blocks of some sequences, end to end
    int j0 = 0, end = 0;
    if (b0 + int(threadIdx.x) < c.batch) filled_blocks(a, b0 + int(threadIdx.x), j0, end);
    int upto = end - j0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    __syncthreads();  // the sequences before have been read
    if (lane == 31) s_sum[warp] = upto;
    s_first[threadIdx.x] = j0;
    __syncthreads();
    int blocks = 0;
#pragma unroll
    for (int w = 0; w < kIndexWarps; ++w) {
      if (w < warp) upto += s_sum[w];
      blocks += s_sum[w];
    }
    s_from[threadIdx.x] = upto - (end - j0);
    __syncthreads();
    int from[kSeqs / 32];
#pragma unroll
    for (int i = 0; i < kSeqs / 32; ++i) from[i] = s_from[i * 32 + lane];
    // the warp's k-th piece: of block block0 + (k >> pieces_log2) * stride; its page, or one outside the pool
    auto find = [&](int k, int& j) {
      const int block = block0 + (k >> pieces_log2) * stride;
      int of = -1;  // the last sequence that starts at or before it
#pragma unroll
      for (int i = 0; i < kSeqs / 32; ++i) of += __popc(__ballot_sync(0xffffffffu, from[i] <= block));
      j = s_first[of] + block - s_from[of];
      return c.tables[(b0 + of) * c.table_stride + (j >> pl)];
    };
    auto issue = [&](int k, int stage) {
      int j;
      const int page = find(k, j);
      if (lane == 0) {
        if (unsigned(page) < unsigned(c.num_pages))
          sm100::mbar_arrive_expect_tx(bars + stage, P::kTiles * P::kTile);
        else
          sm100::mbar_arrive(bars + stage);
      }
      __syncwarp();
      if (unsigned(page) < unsigned(c.num_pages) && lane < 2 * P::kTiles) {
        const int tile = ((j & (per_page - 1)) << (a.block_log2 - 4)) + (k & ((1 << pieces_log2) - 1)) * P::kTiles + (lane >> 1);
        const uint8_t* from = c.pool + page * c.page_stride + ((int64_t(h) << (c.page_log2 - 4)) + tile) * L.bytes();
        uint8_t* to = stages + stage * P::kBytes + (lane >> 1) * P::kTile;
        if (lane & 1)
          bulk_g2s(to + P::kCodes, from + L.k_scales(), P::kRest, bars + stage);
        else
          bulk_g2s(to, from + L.k_codes(), P::kCodes, bars + stage);
      }
    };
    auto arrived = [&](int stage, uint32_t parity) {  // (the vote makes the lanes agree)
      const bool ok = __all_sync(0xffffffffu, sm100::mbar_wait(bars + stage, parity, &s_never));
      if (!ok && lane == 0) atomicAdd(&g_paged_index_timeouts, 1);
      return ok;
    };
    ring.start(block0 < blocks ? ((blocks - block0 + stride - 1) / stride) << pieces_log2 : 0, issue);
    Range r;
    for (int k = 0; ring.more(); ++k) {
      if (!ring.take(arrived)) break;  // (a copy that did not arrive: counted, the index is undefined)
      int j;
      const int page = find(k, j);
      const bool held = unsigned(page) < unsigned(c.num_pages);
      if ((k & ((1 << pieces_log2) - 1)) == 0) r.clear();
      if (held) {
        const uint8_t* piece = stages + ring.stage * P::kBytes;
#pragma unroll 1
        for (int x = 0; x < P::kTiles; ++x, piece += P::kTile) {
          const uint32_t* codes = reinterpret_cast<const uint32_t*>(piece) + at.row * W + at.word;
          const __half* scales = reinterpret_cast<const __half*>(piece + P::kCodes) + at.row * G + at.g;
          const uint8_t* zeros = piece + P::kCodes + (L.k_zeros() - L.k_scales()) + at.row * G + at.g;
#pragma unroll
          for (int t = 0; t < 16; t += 2 * ROWS) {
            if constexpr (ROWS == 8) {  // one token a lane in half a tile: the two halves
              r.add({codes[0], codes[8 * W]}, {__half2float(scales[0]), __half2float(scales[8 * G])},
                    {float(zeros[0]), float(zeros[8 * G])}, e12, e16);
            } else {
              const int u = t + ROWS;
              r.add({codes[t * W], codes[u * W]}, {__half2float(scales[t * G]), __half2float(scales[u * G])},
                    {float(zeros[t * G]), float(zeros[u * G])}, e12, e16);
            }
          }
        }
      }
      __syncwarp();
      ring.next(issue);
      if (held && ((k + 1) & ((1 << pieces_log2) - 1)) == 0) {
        at.join_rows(r);
        at.store(a, (int64_t(page) * c.kv_heads + h) * per_page + (j & (per_page - 1)), r,
                 __any_sync(0xffffffffu, !(r.finite == 0.f)), lane);
      }
    }
  }
}

template <int G>
int launch_index(const PagedIndexArgs& a, cudaStream_t st) {
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  constexpr int kSmem = Piece<G>::kSmem;
  e = once.run(dev, [&] { return cudaFuncSetAttribute(paged_index_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); });
  if (e != cudaSuccess) return cuda_status(e);
  // a sequence's new tokens fill at most this many blocks (more, where the host's bound does not hold: the kernels loop)
  const int64_t blocks = (int64_t(a.c.max_q) + (1 << a.block_log2) - 1) >> a.block_log2;
  const int64_t items = blocks * a.c.kv_heads, sms = device_sms(dev);
  // (A token or a few of many sequences: most fill no block, and a CTA that finds that out leaves at once.  Measured, one
  // token each, 8 heads of 128, a 64th of the sequences fill a block: 512 sequences 5.7 us, with the other kernel 15.9;
  // 4096 sequences 35.2 and 122; 1024 with 32 heads 35.1 and 34.  Where every sequence brings a block of 64 tokens: 14.3
  // and 31.6; 107 and 276; 106 and 120.)
  const bool few = blocks == 1 || items * a.c.batch <= 16 * sms;
  // enough warps to fill the GPU, some blocks each
  const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(sms * Piece<G>::kCtas / a.c.kv_heads, blocks * a.c.batch / kIndexWarps));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = few ? dim3(unsigned(items), unsigned(std::min(a.c.batch, 65535))) : dim3(unsigned(ctas), unsigned(a.c.kv_heads));
  cfg.blockDim = dim3(32 * kIndexWarps);
  cfg.dynamicSmemBytes = few ? 0 : kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, few ? paged_index_few_kernel<G> : paged_index_kernel<G>, a));
}

// ------------------------------------------------------------ choice
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 16;      // blocks whose scores a warp finds at once
constexpr int kMaxTokens = 32;  // of a CTA

// A score's place in the order of unsigned numbers (finite or infinite; never 0).
__device__ __forceinline__ uint32_t order_of(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kAlways = 0xFFFFFFFFu;

struct TakeScratch {
  int hist[256];
  int digit, left, exact;
  int above[kWarps], equal[kWarps];
  uint32_t any[kWarps], every[kWarps];
};

// The `count` largest of keys[0 .. n) that are not 0, the lowest index first among
// equal ones, in ascending order of index, then -1.  By the W threads of a warp or a CTA.
template <int W>
__device__ __forceinline__ void take_best(const uint32_t* keys, int n, int count, int* out, TakeScratch& s) {
  constexpr int WARPS = W / 32;
  const int tid = threadIdx.x % W, warp = tid >> 5, lane = tid & 31;
  auto sync = [] {
    if constexpr (W == 32)
      __syncwarp();
    else
      __syncthreads();
  };
  // the keys to rank: how many, and the bits that not all of them share
  auto ranked = [](uint32_t k) { return k - 1u < kAlways - 1u; };
  int always = 0, others = 0;
  uint32_t any = 0, every = ~0u;
  for (int j = tid; j < n; j += W) {
    const uint32_t k = keys[j];
    always += k == kAlways;
    if (ranked(k)) {
      ++others;
      any |= k;
      every &= k;
    }
  }
  always = __reduce_add_sync(0xffffffffu, always);
  others = __reduce_add_sync(0xffffffffu, others);
  any = __reduce_or_sync(0xffffffffu, any);
  every = __reduce_and_sync(0xffffffffu, every);
  if constexpr (WARPS > 1) {
    if (lane == 0) {
      s.above[warp] = always;
      s.equal[warp] = others;
      s.any[warp] = any;
      s.every[warp] = every;
    }
    sync();
    always = others = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      always += s.above[w];
      others += s.equal[w];
      any |= s.any[w];
      every &= s.every[w];
    }
  }
  // digit by digit, from the first bit that differs: the prefix of the last key to take
  int left = count - always;  // to take among the keys of the prefix
  bool all = others <= left || left == 0;  // ... which is all of them, or none
  const int top = 31 - __clz((any ^ every) | 1);
  uint32_t mask = ~((2u << top) - 1u), prefix = left == 0 ? kAlways : all ? 0 : every & mask;
  for (int shift = max(top - 7, 0), more = 1; more && !all; more = shift > 0, shift = max(shift - 8, 0)) {
    for (int i = tid; i < 256; i += W) s.hist[i] = 0;
    sync();
    for (int j = tid; j < n; j += W) {
      const uint32_t k = keys[j];
      if (ranked(k) && (k & mask) == prefix) atomicAdd(s.hist + (k >> shift & 255u), 1);
    }
    sync();
    if (warp == 0) {  // lane l: digits 255 - 8 l .. 248 - 8 l
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mine[i] = s.hist[255 - 8 * lane - i];
        sum += mine[i];
      }
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      before -= sum;
      if (before < left && left <= before + sum) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < left && left <= before + mine[i]) {
            s.digit = 255 - 8 * lane - i;
            s.left = left - before;
            s.exact = mine[i] == left - before;
          }
          before += mine[i];
        }
      }
    }
    sync();
    prefix |= uint32_t(s.digit) << shift;  // (digits overlap where the last one is cut: the bits are the same)
    mask |= 255u << shift;
    left = s.left;
    all = s.exact != 0;
  }
  if constexpr (WARPS > 1) sync();
  // taken: above the threshold, and `left` that equal it
  const uint32_t least = all ? max(prefix, 1u) : prefix;  // all: every key from here on is taken
  if (all) left = 0;
  auto above = [&](uint32_t k) { return all ? k >= least : k > least; };
  const int span = (n + W - 1) / W * 32, from = warp * span, to = min(n, from + span);
  int taken = 0, equal = 0, whole = left;
  if constexpr (WARPS > 1) {
    int n_above = 0, n_equal = 0;
    for (int j0 = from; j0 < to; j0 += 32) {
      const uint32_t k = j0 + lane < to ? keys[j0 + lane] : 0;
      n_above += __popc(__ballot_sync(0xffffffffu, k && above(k)));
      n_equal += __popc(__ballot_sync(0xffffffffu, !all && k == least));
    }
    if (lane == 0) {
      s.above[warp] = n_above;
      s.equal[warp] = n_equal;
    }
    sync();
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) {
        taken += s.above[w];
        equal += s.equal[w];
      }
      whole += s.above[w];
    }
  }
  for (int j0 = from; j0 < to; j0 += 32) {
    const uint32_t k = j0 + lane < to ? keys[j0 + lane] : 0;
    const uint32_t ups = __ballot_sync(0xffffffffu, k && above(k)), eqs = __ballot_sync(0xffffffffu, !all && k == least);
    const uint32_t below = (1u << lane) - 1;
    const int at_above = taken + __popc(ups & below), at_equal = equal + __popc(eqs & below);
    if (ups >> lane & 1u) out[at_above + min(at_equal, left)] = j0 + lane;
    else if ((eqs >> lane & 1u) && at_equal < left) out[at_above + at_equal] = j0 + lane;
    taken += __popc(ups);
    equal += __popc(eqs);
  }
  if constexpr (WARPS == 1) whole += taken;
  for (int i = whole + tid; i < count; i += W) out[i] = -1;
  sync();
}

// D += A B of mma.sync m16n8k32, s8 in, s32 out.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct SelectParams {
  PagedSelectArgs a;
  int tokens;  // of a CTA
  int pitch;   // keys of a token
};

// Measured: one token, 2048 blocks, 8 heads of 128 (a cluster of 8 CTAs a list) 10.5 to 11.4 us,
// most of it a chain of look-ups, two cluster barriers and the ranking; 64 ragged sequences of up to 256
// blocks 10.7 us (19.7 MB of index: 1.8 TB/s); 512 tokens over 512 blocks (8 tokens a CTA) 46 us, where the
// ranking by single warps takes as many instructions as the scores.
//
// A cluster has one key/value head and `tokens` new tokens in a row, its CTAs every
// n-th tile of 16 blocks; the first CTA keeps the keys and takes the best.  Columns of
// the products: query heads of the tokens, 8 NT at a time.  Operand A, 16 blocks x 32
// bytes of codes: lane (g, c) has bytes 16 c .. of a 64-byte piece of blocks g and g + 8
// as they lie in memory, so the k index runs differently than the bytes, the same way in
// operand B.
template <int G, int NT>
__global__ void __launch_bounds__(kThreads, G < 8 ? (NT == 1 ? 4 : 2) : 2) paged_select_kernel(SelectParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  sm100::pdl_wait();
  sm100::pdl_trigger();
  constexpr int D = 32 * G, COLS = 8 * NT;
  const PagedSelectArgs& a = p.a;
  const PagedView& c = a.i.c;
  extern __shared__ __align__(16) uint8_t smem[];
  int8_t* frag = reinterpret_cast<int8_t*>(smem);                     // [G][NT][32 lanes][16 bytes]
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem + G * NT * 512);  // [tokens][pitch]
  __shared__ TakeScratch s_take[kWarps];
  __shared__ int s_pos[kMaxTokens], s_seq[kMaxTokens];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int h = blockIdx.x / ctas, bl = a.i.block_log2, pl = c.page_log2 - bl, per_page = 1 << pl;
  uint32_t* best = ctas > 1 ? cluster.map_shared_rank(keys, 0) : keys;

  for (int64_t t0 = int64_t(blockIdx.y) * p.tokens; t0 < c.total; t0 += int64_t(gridDim.y) * p.tokens) {
    const int tokens = int(c.total - t0 < p.tokens ? c.total - t0 : p.tokens);
    // ---- sequences and positions (-1: no place in the cache)
    for (int i = warp; i < tokens; i += kWarps) {
      const int64_t t = t0 + i;
      const int b = sequence_of(c, t);
      int pos = -1;
      if (b >= 0) {
        int64_t first;
        int count;
        new_tokens(c, b, first, count);
        pos = c.seq_lens[b] - count + int(t - first);
        if (pos >= c.limit) pos = -1;
      }
      if (lane == 0) {
        s_pos[i] = pos;
        s_seq[i] = b;
      }
    }
    __syncthreads();
    if (rank == 0) {
      for (int i = 0; i < tokens; ++i) {
        const int n = s_pos[i] < 0 ? 0 : (s_pos[i] >> bl) + 1;
        for (int j = tid; j < n; j += kThreads) {
          // those that are always taken (scores never touch their keys)
          const bool always = n <= a.count || j < a.first || j >= n - a.last;
          const int page = always ? c.tables[s_seq[i] * c.table_stride + (j >> pl)] : -1;
          keys[i * p.pitch + j] = unsigned(page) < unsigned(c.num_pages) ? kAlways : 0;
        }
      }
    }
    if (ctas > 1) cluster.sync(); else __syncthreads();

    // ---- scores, one run of tokens of the same sequence after the other
    for (int i0 = 0, i1; i0 < tokens; i0 = i1) {
      const int b = s_seq[i0];
      int n = 0;  // blocks that a token of the run chooses among
      for (i1 = i0; i1 < tokens && s_seq[i1] == b; ++i1) {
        const int of = s_pos[i1] < 0 ? 0 : (s_pos[i1] >> bl) + 1;
        if (of > a.count) n = max(n, of - a.last);
      }
      if (n == 0) continue;
      const int* table = c.tables + b * c.table_stride;
      const int columns = (i1 - i0) * a.group;
      for (int col0 = 0; col0 < columns; col0 += COLS) {
        __syncthreads();  // the fragments of the columns before have been used
        for (int i = warp; i < COLS; i += kWarps) {
          // four features a lane: d = 4 lane .. of every 128
          constexpr int R = (G + 3) / 4;
          const int col = col0 + i;
          float x[4 * R], top = 0.f;
          bool bad = false;
#pragma unroll
          for (int k = 0; k < 4 * R; ++k) x[k] = 0.f;
          if (col < columns) {
            const int tok = col / a.group, head = h * a.group + col - tok * a.group;
            const uint16_t* from = reinterpret_cast<const uint16_t*>(a.q) + (t0 + i0 + tok) * a.q_ts + head * a.q_hs + 4 * lane;
#pragma unroll
            for (int k = 0; k < R; ++k) {
              if (k * 128 + 4 * lane >= D) continue;
              uint2 w;
              if (a.vec) {
                w = __ldcg(reinterpret_cast<const uint2*>(from + k * 128));
              } else {
                w.x = uint32_t(__ldcg(from + k * 128)) | uint32_t(__ldcg(from + k * 128 + 1)) << 16;
                w.y = uint32_t(__ldcg(from + k * 128 + 2)) | uint32_t(__ldcg(from + k * 128 + 3)) << 16;
              }
#pragma unroll
              for (int z = 0; z < 4; ++z) x[4 * k + z] = bits_to_float((z < 2 ? w.x : w.y) >> (16 * (z & 1)) & 0xFFFFu, a.dtype);
            }
#pragma unroll
            for (int k = 0; k < 4 * R; ++k) {
              bad = bad || !(fabsf(x[k]) < INFINITY);
              top = fmaxf(top, fabsf(x[k]));
            }
          }
          bad = __any_sync(0xffffffffu, bad);
          // (magnitudes, as whole numbers in the order of the values)
          top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
          const float inv = inverse_step(range_step(bad ? 0.f : top));
#pragma unroll
          for (int k = 0; k < R; ++k) {
            if (k * 128 + 4 * lane >= D) continue;
            uint32_t up = 0, down = 0;  // codes above 0 for the largest values, below 0 for the smallest
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int code = bad ? 0 : int(rintf(x[4 * k + z] * inv));
              up |= uint32_t(max(code, 0)) << (8 * z);
              down |= (uint32_t(min(code, 0)) & 255u) << (8 * z);
            }
            auto put = [&](int d, uint32_t w) {
              *reinterpret_cast<uint32_t*>(frag + (((d >> 6) * NT + (i >> 3)) * 32 + (i & 7) * 4 + (d >> 4 & 3)) * 16 + (d & 15)) = w;
            };
            put(k * 128 + 4 * lane, up);
            put(D + k * 128 + 4 * lane, down);
          }
        }
        __syncthreads();
        // of a lane's columns (or of those it speaks for): where their token's keys are, and for how many blocks
        constexpr int NV = 2 * NT;
        int at[NV], below[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = col0 + (i >> 1) * 8 + 2 * cc + (i & 1);
          const bool silent = (a.group % 2 == 0 && (i & 1)) || (a.group % 4 == 0 && (cc & 1)) || (a.group % 8 == 0 && (cc & 2));
          at[i] = below[i] = 0;
          if (col < columns && !silent) {
            const int tok = i0 + col / a.group, m = (s_pos[tok] >> bl) + 1;
            at[i] = tok * p.pitch;
            if (m > a.count) below[i] = m - a.last;
          }
        }
        for (int j0 = (warp * ctas + rank) * kTile; j0 < n; j0 += kWarps * ctas * kTile) {
          uint4 k0[G], k1[G];
          float s0 = 0.f, s1 = 0.f;
          bool in0 = false, in1 = false;
          auto load = [&](int j, uint4 (&k)[G], float& s, bool& in) {
            const int page = j < n && j >= a.first ? table[j >> pl] : -1;
            in = unsigned(page) < unsigned(c.num_pages);
            const int64_t slot = (int64_t(in ? page : 0) * c.kv_heads + h) * per_page + (j & (per_page - 1));
            const uint4* from = reinterpret_cast<const uint4*>(a.i.codes + slot * 2 * D) + cc;
#pragma unroll
            for (int i = 0; i < G; ++i) k[i] = in ? __ldcg(from + 4 * i) : make_uint4(0, 0, 0, 0);
            if (in) s = __ldcg(a.i.scales + slot);
          };
          load(j0 + g, k0, s0, in0);
          load(j0 + g + 8, k1, s1, in1);
          int d[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[nt][i] = 0;
#pragma unroll
          for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint4 q = reinterpret_cast<const uint4*>(frag)[(i * NT + nt) * 32 + lane];
              mma_s8(d[nt], k0[i].x, k1[i].x, k0[i].y, k1[i].y, q.x, q.y);
              mma_s8(d[nt], k0[i].z, k1[i].z, k0[i].w, k1[i].w, q.z, q.w);
            }
          }
          // the best head of each token: columns of a lane, of its neighbours, then in shared memory
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int j = j0 + g + 8 * half;
              int v0 = d[nt][2 * half];
              const int v1 = d[nt][2 * half + 1];
              if (a.group % 2 == 0) v0 = max(v0, v1);  // (a token's columns, or columns of none)
              if (a.group % 4 == 0) v0 = max(v0, __shfl_xor_sync(0xffffffffu, v0, 1));
              if (a.group % 8 == 0) v0 = max(v0, __shfl_xor_sync(0xffffffffu, v0, 2));
              if (!(half ? in1 : in0)) continue;
              const float s = half ? s1 : s0;
              if (j < below[2 * nt]) atomicMax(best + at[2 * nt] + j, order_of(s < INFINITY ? float(v0) * s : INFINITY));
              if (j < below[2 * nt + 1]) atomicMax(best + at[2 * nt + 1] + j, order_of(s < INFINITY ? float(v1) * s : INFINITY));
            }
          }
        }
      }
    }
    // ---- the best
    if (ctas > 1) cluster.sync(); else __syncthreads();
    if (rank == 0) {
      if (p.tokens == 1) {
        take_best<kThreads>(keys, s_pos[0] < 0 ? 0 : (s_pos[0] >> bl) + 1, a.count, a.blocks + t0 * a.b_ts + h * a.b_hs, s_take[0]);
      } else {
        for (int i = warp; i < tokens; i += kWarps)
          take_best<32>(keys + i * p.pitch, s_pos[i] < 0 ? 0 : (s_pos[i] >> bl) + 1, a.count,
                        a.blocks + (t0 + i) * a.b_ts + h * a.b_hs, s_take[warp]);
      }
    }
    __syncthreads();
    if (ctas > 1) cluster.sync();  // before the keys are cleared
  }
}

template <int G, int NT>
int launch_select_as(const PagedSelectArgs& a, int tokens, int ctas, cudaStream_t st) {
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  auto kern = paged_select_kernel<G, NT>;
  constexpr int kFrag = G * NT * 512;
  e = once.run(dev, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFrag + SPECTRA_MAX_INDEXED_BLOCKS * 4);
  });
  if (e != cudaSuccess) return cuda_status(e);
  SelectParams p;
  p.a = a;
  p.tokens = tokens;
  p.pitch = a.max_blocks;
  const int64_t groups = (a.i.c.total + tokens - 1) / tokens;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.i.c.kv_heads * ctas), unsigned(std::min<int64_t>(groups, 65535)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(kFrag) + size_t(tokens) * p.pitch * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

template <int G>
int launch_select(const PagedSelectArgs& a, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  const int64_t sms = device_sms(dev), lists = a.i.c.total * a.i.c.kv_heads;
  // Prompts: several tokens a CTA, up to 32 columns, so that codes are read once for all of them; fewer while their
  // CTAs still run at once (four an SM with up to 8 columns, else two), and while two CTAs' keys do not fit an SM.
  // Measured, heads of 128, 32 or 64 query heads on 8: 128 tokens over 32768 with 2 tokens a CTA 20.7 us, with 4 22.0
  // (64 heads: 38.7, and with 4, at once, 23.8); 256 tokens with 4 39.9, with 8, at once, 25.9; 512 tokens with 8 47.9,
  // with 4 76.8; 64 tokens of 64 heads with one 18.0, with 2 20.2 (32 heads: 17.9 and 15.9).  8 tokens with 2048 blocks
  // each take 131 us for 512 tokens over 131072, 4 of them 219.
  int tokens = std::min({32 / a.group, kMaxTokens, a.i.c.max_q});
  auto at_once = [&](int n) { return sms * (G < 8 && n * a.group <= 8 ? 4 : 2); };
  while (tokens > 1 && (int64_t(tokens) * a.max_blocks > 24 * 1024 || lists <= at_once(tokens / 2) * (tokens / 2))) tokens /= 2;
  if (tokens > 1) return tokens * a.group <= 8 ? launch_select_as<G, 1>(a, tokens, 1, st) : launch_select_as<G, 4>(a, tokens, 1, st);
  // Few lists: several CTAs each, while they have a tile for every warp.
  int ctas = 1;
  while (ctas < 8 && lists * ctas < sms && a.max_blocks > 2 * ctas * kWarps * kTile) ctas *= 2;
  return a.group <= 8 ? launch_select_as<G, 1>(a, 1, ctas, st) : launch_select_as<G, 4>(a, 1, ctas, st);
}

}  // namespace

int launch_paged_index(const PagedIndexArgs& a, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 32: return launch_index<1>(a, st);
    case 64: return launch_index<2>(a, st);
    case 96: return launch_index<3>(a, st);
    case 128: return launch_index<4>(a, st);
    case 256: return launch_index<8>(a, st);
  }
  return SPECTRA_ERR_UNSUPPORTED;
}

int paged_index_timeouts(long long* out, bool reset) { return read_timeout_counter(g_paged_index_timeouts, out, reset); }

int launch_paged_select(const PagedSelectArgs& a, cudaStream_t st) {
  switch (a.i.c.head_dim) {
    case 32: return launch_select<1>(a, st);
    case 64: return launch_select<2>(a, st);
    case 96: return launch_select<3>(a, st);
    case 128: return launch_select<4>(a, st);
    case 256: return launch_select<8>(a, st);
  }
  return SPECTRA_ERR_UNSUPPORTED;
}

}  // namespace spectra
