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
// an upper bound of every c_h . k of the block, up to S's rounding.  The sum is
// max(c, 0) . H + min(c, 0) . L, a product of integers below 2^22, so scores are
// exact in fp32 and the choice does not depend on the order of the sums.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

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
// -(2048 + z) s or -(128 + z) s makes it (q - z) s: 23 and 19 bits, exact.  Bound by these
// instructions.
constexpr int kIndexWarps = 4;  // of a CTA
constexpr int kIndexTokens = 16;

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

// SPLIT: warps that share a block (1, or all of the CTA).
template <int G, int SPLIT>
__global__ void __launch_bounds__(32 * kIndexWarps) paged_index_kernel(PagedIndexArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  constexpr int D = 32 * G, W = 4 * G, ROWS = G == 8 ? 1 : G >= 3 ? 2 : 8 / G;
  constexpr int AT_ONCE = SPLIT > 1 ? 8 : kIndexTokens;  // tokens of a warp whose loads are in flight
  constexpr int FLIGHT = AT_ONCE / ROWS;
  constexpr TileLayout L{G};
  const PagedView& c = a.c;
  __shared__ float2 s_part[SPLIT > 1 ? SPLIT : 1][8][SPLIT > 1 ? W : 1];  // [warp][feature of a word][word]: largest, smallest
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = min(lane / W, ROWS - 1), word = lane < ROWS * W ? lane % W : 0;
  const int g = word % G, d0 = g * 32 + word / G * 8;  // its features d0 .. d0 + 7
  const int to_word = (row * W + word) * 4, to_scale = (row * G + g) * 2, to_zero = row * G + g;
  const uint32_t e12 = in_register(0x45000000u), e16 = in_register(0x43000000u);
  const int pl = c.page_log2 - a.block_log2, per_page = 1 << pl, tiles = 1 << (a.block_log2 - 4);
  for (int b = blockIdx.y; b < c.batch; b += gridDim.y) {
    int64_t first;
    int count;
    new_tokens(c, b, first, count);
    const int held = c.seq_lens[b], len = min(held, c.limit);
    if (len <= 0 || count == 0) continue;
    const int j0 = max(held - count, 0) >> a.block_log2, end = len >> a.block_log2;
    constexpr int AT_A_TIME = kIndexWarps / SPLIT;  // blocks of a CTA
    for (int64_t item = int64_t(blockIdx.x) * AT_A_TIME + warp / SPLIT; item < int64_t(end - j0) * c.kv_heads;
         item += int64_t(gridDim.x) * AT_A_TIME) {
      const int j = j0 + int(item / c.kv_heads), h = int(item % c.kv_heads);
      const int page = c.tables[b * c.table_stride + (j >> pl)];
      if (unsigned(page) >= unsigned(c.num_pages)) continue;
      const int part = j & (per_page - 1);
      const uint8_t* t = c.pool + page * c.page_stride +
                         ((int64_t(h) << (c.page_log2 - 4)) + int64_t(part) * tiles) * L.bytes();
      float hi[8], lo[8], finite = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = -INFINITY;
        lo[i] = INFINITY;
      }
      const int share = tiles * 16 / SPLIT, k_end = warp % SPLIT * share + share;
      for (int k0 = k_end - share; k0 < k_end; k0 += AT_ONCE) {
        // (a flight of 8 tokens is half a tile)
        const uint8_t* from = t + (k0 >> 4) * L.bytes();
        const int half = AT_ONCE == 8 ? k0 >> 3 & 1 : 0;
        uint32_t w[FLIGHT];
        __half s16[FLIGHT];
        uint8_t z8[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
          const int tok = k * ROWS;  // (and row)
          const uint8_t* tile = from + (tok >> 4) * L.bytes();
          w[k] = __ldcg(reinterpret_cast<const uint32_t*>(tile + L.k_codes() + (half + (tok >> 3 & 1)) * L.block() + (tok & 7) * W * 4 + to_word));
          s16[k] = __ldcg(reinterpret_cast<const __half*>(tile + L.k_scales() + (8 * half + (tok & 15)) * G * 2 + to_scale));
          z8[k] = __ldcg(tile + L.k_zeros() + (8 * half + (tok & 15)) * G + to_zero);
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; k += 2) {
          float v[2][8];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float s = __half2float(s16[k + x]), z = float(z8[k + x]);
            const float c12 = -(2048.f + z) * s, c16 = -(128.f + z) * s;
            finite = fmaf(s, 0.f, finite);
            const uint32_t q[4] = {w[k + x] << 12, w[k + x] << 4, w[k + x] >> 4, w[k + x] >> 12};
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
      }
      // the rows: lanes of the same word, then every word's largest magnitude
#pragma unroll
      for (int o = W; o < ROWS * W; o *= 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hi[i] = fmaxf(hi[i], __shfl_down_sync(0xffffffffu, hi[i], o));
          lo[i] = fminf(lo[i], __shfl_down_sync(0xffffffffu, lo[i], o));
        }
      }
      bool bad = __any_sync(0xffffffffu, !(finite == 0.f));
      if constexpr (SPLIT > 1) {
        if (lane < W) {
#pragma unroll
          for (int i = 0; i < 8; ++i) s_part[warp][i][lane] = make_float2(hi[i], lo[i]);
        }
        bad = __syncthreads_or(bad);
        if (warp == 0 && lane < W) {
#pragma unroll
          for (int x = 1; x < SPLIT; ++x)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              hi[i] = fmaxf(hi[i], s_part[x][i][lane].x);
              lo[i] = fminf(lo[i], s_part[x][i][lane].y);
            }
        }
        __syncthreads();  // before the next block's are written
        if (warp > 0) continue;
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
      // (magnitudes, as whole numbers in the order of the values; of the lanes that hold all rows)
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < W && !bad ? __float_as_uint(top) : 0u));
      const float step = range_step(top), inv = inverse_step(step);
      const int64_t slot = (int64_t(page) * c.kv_heads + h) * per_page + part;
      if (lane < W) {
        uint32_t up[2] = {0, 0}, down[2] = {0, 0};
        if (!bad) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            up[i >> 2] |= (uint32_t(int(ceilf(hi[i] * inv))) & 255u) << (8 * (i & 3));
            down[i >> 2] |= (uint32_t(int(floorf(lo[i] * inv))) & 255u) << (8 * (i & 3));
          }
        }
        *reinterpret_cast<uint2*>(a.codes + slot * 2 * D + d0) = make_uint2(up[0], up[1]);
        *reinterpret_cast<uint2*>(a.codes + slot * 2 * D + D + d0) = make_uint2(down[0], down[1]);
      }
      if (lane == 0) a.scales[slot] = bad ? INFINITY : step;
    }
  }
}

template <int G>
int launch_index(const PagedIndexArgs& a, cudaStream_t st) {
  // a sequence's new tokens fill at most this many blocks (more, where the host's bound does not hold: the kernel loops)
  const int64_t blocks = (int64_t(a.c.max_q) + (1 << a.block_log2) - 1) >> a.block_log2;
  const int64_t items = blocks * a.c.kv_heads;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  // few blocks: four warps each
  const bool split = items * a.c.batch <= 16 * device_sms(dev);
  const int64_t ctas = split ? items : (items + kIndexWarps - 1) / kIndexWarps;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(ctas, INT32_MAX)), unsigned(std::min(a.c.batch, 65535)));
  cfg.blockDim = dim3(32 * kIndexWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, split ? paged_index_kernel<G, kIndexWarps> : paged_index_kernel<G, 1>, a));
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
  // Prompts: several tokens a CTA, up to 32 columns, so that codes are read once for all of them.
  int tokens = std::min({32 / a.group, kMaxTokens, a.i.c.max_q});
  while (tokens > 1 && (int64_t(tokens) * a.max_blocks > 24 * 1024 || lists < 2 * sms * tokens)) tokens /= 2;
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
