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
constexpr int kRowsAtOnce = 8;  // tokens that a CTA reads at once: half a tile

template <int G>
__global__ void __launch_bounds__(32 * G) paged_index_kernel(PagedIndexArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  constexpr int D = 32 * G, W = 4 * G;
  constexpr TileLayout L{G};
  __shared__ float4 s_hi[kRowsAtOnce * W * 2], s_lo[kRowsAtOnce * W * 2];
  __shared__ float s_top[G];
  const PagedView& c = a.c;
  const int tid = threadIdx.x, row = tid / W, word = tid - row * W, g = word % G;
  const int h = blockIdx.x, per_page = 1 << (c.page_log2 - a.block_log2), tiles = 1 << (a.block_log2 - 4);
  for (int b = blockIdx.z; b < c.batch; b += gridDim.z) {
    int64_t first;
    int count;
    new_tokens(c, b, first, count);
    const int held = c.seq_lens[b], len = min(held, c.limit);
    if (len <= 0 || count == 0) continue;
    const int end = len >> a.block_log2;
    for (int j = (max(held - count, 0) >> a.block_log2) + int(blockIdx.y); j < end; j += gridDim.y) {
      const int page = c.tables[b * c.table_stride + (j >> (c.page_log2 - a.block_log2))];
      if (unsigned(page) >= unsigned(c.num_pages)) continue;
      const int part = j & (per_page - 1);
      const uint8_t* t = c.pool + page * c.page_stride +
                         ((int64_t(h) << (c.page_log2 - 4)) + int64_t(part) * tiles) * L.bytes();
      float hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = -INFINITY;
        lo[i] = INFINITY;
      }
      bool bad = false;
#pragma unroll 4
      for (int k = 0; k < 2 * tiles; ++k) {
        const uint8_t* tile = t + (k >> 1) * L.bytes();
        const int tok = (k & 1) * 8 + row;
        const uint32_t w = reinterpret_cast<const uint32_t*>(tile + L.k_codes() + (k & 1) * L.block())[tid];
        const float s = __half2float(reinterpret_cast<const __half*>(tile + L.k_scales())[tok * G + g]);
        const float z = float(tile[L.k_zeros() + tok * G + g]);
        bad = bad || !(fabsf(s) <= 65504.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = (float((w >> (4 * i)) & 15u) - z) * s;
          hi[i] = fmaxf(hi[i], v);
          lo[i] = fminf(lo[i], v);
        }
      }
      float4* out = s_hi + tid * 2;
      out[0] = make_float4(hi[0], hi[1], hi[2], hi[3]);
      out[1] = make_float4(hi[4], hi[5], hi[6], hi[7]);
      out = s_lo + tid * 2;
      out[0] = make_float4(lo[0], lo[1], lo[2], lo[3]);
      out[1] = make_float4(lo[4], lo[5], lo[6], lo[7]);
      bad = __syncthreads_or(bad);
      // thread d: feature d = word (d % 32) / 8 of group d / 32, its d % 8-th
      const int at = (((tid & 31) >> 3) * G + (tid >> 5)) * 8 + (tid & 7);
      float up = -INFINITY, down = INFINITY;
#pragma unroll
      for (int i = 0; i < kRowsAtOnce; ++i) {
        up = fmaxf(up, reinterpret_cast<const float*>(s_hi)[i * W * 8 + at]);
        down = fminf(down, reinterpret_cast<const float*>(s_lo)[i * W * 8 + at]);
      }
      float top = bad ? 0.f : fmaxf(fabsf(up), fabsf(down));
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((tid & 31) == 0) s_top[tid >> 5] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < G; ++i) top = fmaxf(top, s_top[i]);
      const float step = range_step(top), inv = inverse_step(step);
      const int64_t slot = (int64_t(page) * c.kv_heads + h) * per_page + part;
      int8_t* codes = a.codes + slot * 2 * D;
      codes[tid] = bad ? 0 : int8_t(int(ceilf(up * inv)));
      codes[D + tid] = bad ? 0 : int8_t(int(floorf(down * inv)));
      if (tid == 0) a.scales[slot] = bad ? INFINITY : step;
      __syncthreads();  // before the next block writes what this one still reads
    }
  }
}

template <int G>
int launch_index(const PagedIndexArgs& a, cudaStream_t st) {
  // a sequence's new tokens fill at most this many blocks (more, where the host's bound does not hold: the kernel loops)
  const int64_t blocks = (int64_t(a.c.max_q) + (1 << a.block_log2) - 1) >> a.block_log2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.c.kv_heads), unsigned(std::min<int64_t>(blocks, 65535)),
                     unsigned(std::min(a.c.batch, 65535)));
  cfg.blockDim = dim3(32 * G);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_index_kernel<G>, a));
}

// ------------------------------------------------------------ choice
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kHeads = 8;  // query heads whose codes are in shared memory at once

// A score's place in the order of unsigned numbers (finite or infinite; never 0).
__device__ __forceinline__ uint32_t order_of(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kAlways = 0xFFFFFFFFu;

// The `count` largest of keys[0 .. n) that are not 0, the lowest index first among
// equal ones, in ascending order of index, then -1.
__device__ __forceinline__ void take_best(const uint32_t* keys, int n, int count, int* out) {
  __shared__ int s_hist[256];
  __shared__ int s_digit, s_left, s_exact;
  __shared__ int s_above[kWarps], s_equal[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // digit by digit from the top: the prefix of the count-th largest key
  uint32_t prefix = 0, mask = 0;
  int left = count;  // to take among the keys of the prefix
  bool all = false;  // ... which is all of them
  for (int shift = 24; shift >= 0 && !all; shift -= 8) {
    s_hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kThreads) {
      const uint32_t k = keys[j];
      if (k && (k & mask) == prefix) atomicAdd(s_hist + (k >> shift & 255u), 1);
    }
    __syncthreads();
    if (warp == 0) {  // lane l: digits 255 - 8 l .. 248 - 8 l
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mine[i] = s_hist[255 - 8 * lane - i];
        sum += mine[i];
      }
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      const int total = __shfl_sync(0xffffffffu, before, 31);
      before -= sum;
      if (lane == 0 && total <= left) {  // fewer than asked for: all of them
        s_digit = 0;
        s_left = 0;
        s_exact = 2;
      }
      if (total > left && before < left && left <= before + sum) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < left && left <= before + mine[i]) {
            s_digit = 255 - 8 * lane - i;
            s_left = left - before;
            s_exact = mine[i] == left - before;
          }
          before += mine[i];
        }
      }
    }
    __syncthreads();
    if (s_exact == 2) {
      all = true;  // (only in the first round: later ones have enough keys)
    } else {
      prefix |= uint32_t(s_digit) << shift;
      mask |= 255u << shift;
      left = s_left;
      all = s_exact != 0;
    }
    __syncthreads();
  }
  // taken: above the threshold, and `left` that equal it
  const uint32_t least = all ? max(prefix, 1u) : prefix;  // all: every key from here on is taken
  if (all) left = 0;
  auto above = [&](uint32_t k) { return all ? k >= least : k > least; };
  const int span = (n + kThreads - 1) / kThreads * 32, from = warp * span, to = min(n, from + span);
  int n_above = 0, n_equal = 0;
  for (int j0 = from; j0 < to; j0 += 32) {
    const uint32_t k = j0 + lane < to ? keys[j0 + lane] : 0;
    n_above += __popc(__ballot_sync(0xffffffffu, k && above(k)));
    n_equal += __popc(__ballot_sync(0xffffffffu, !all && k == least));
  }
  if (lane == 0) {
    s_above[warp] = n_above;
    s_equal[warp] = n_equal;
  }
  __syncthreads();
  int taken = 0, equal = 0, whole = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      taken += s_above[w];
      equal += s_equal[w];
    }
    whole += s_above[w];
  }
  whole += left;
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
  for (int i = whole + tid; i < count; i += kThreads) out[i] = -1;
}

template <int G>
__global__ void __launch_bounds__(kThreads) paged_select_kernel(PagedSelectArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  constexpr int D = 32 * G, D4 = 2 * D / 4;
  extern __shared__ __align__(16) uint32_t keys[];  // [max_blocks]
  __shared__ __align__(16) int8_t s_code[kHeads][2 * D];
  const PagedView& c = a.i.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x, bl = a.i.block_log2, per_page = 1 << (c.page_log2 - bl);
  for (int64_t t = blockIdx.y; t < c.total; t += gridDim.y) {
    int* out = a.blocks + t * a.b_ts + h * a.b_hs;
    const int b = sequence_of(c, t);
    int pos = -1;
    if (b >= 0) {
      int64_t first;
      int count;
      new_tokens(c, b, first, count);
      pos = c.seq_lens[b] - count + int(t - first);
      if (pos >= c.limit) pos = -1;
    }
    if (pos < 0) {
      for (int i = tid; i < a.count; i += kThreads) out[i] = -1;
      continue;
    }
    const int n = (pos >> bl) + 1;
    const int* table = c.tables + b * c.table_stride;
    const bool scored = n > a.count;
    int* sums = reinterpret_cast<int*>(keys);
    for (int j = tid; j < n; j += kThreads) sums[j] = INT32_MIN;
    for (int g0 = 0; g0 < a.group && scored; g0 += kHeads) {
      const int heads = min(kHeads, a.group - g0);
      __syncthreads();
      for (int i = warp; i < heads; i += kWarps) {
        const int64_t at = t * a.q_ts + int64_t(h * a.group + g0 + i) * a.q_hs;
        float x[G], top = 0.f;
        bool bad = false;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          x[g] = load_as_float_cg(a.q, at + g * 32 + lane, a.dtype);
          bad = bad || !(fabsf(x[g]) < INFINITY);
          top = fmaxf(top, fabsf(x[g]));
        }
        bad = __any_sync(0xffffffffu, bad);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float inv = inverse_step(range_step(bad ? 0.f : top));
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int code = bad ? 0 : int(rintf(x[g] * inv));
          s_code[i][g * 32 + lane] = int8_t(max(code, 0));
          s_code[i][D + g * 32 + lane] = int8_t(min(code, 0));
        }
      }
      __syncthreads();
      for (int j = a.first + tid; j < n - a.last; j += kThreads) {
        const int page = table[j >> (c.page_log2 - bl)];
        if (unsigned(page) >= unsigned(c.num_pages)) continue;
        const int64_t slot = (int64_t(page) * c.kv_heads + h) * per_page + (j & (per_page - 1));
        const int4* codes = reinterpret_cast<const int4*>(a.i.codes + slot * 2 * D);
        int sum[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) sum[i] = 0;
        for (int w = 0; w < D4 / 4; ++w) {
          const int4 k = codes[w];
#pragma unroll
          for (int i = 0; i < kHeads; ++i) {
            const int4 q = reinterpret_cast<const int4*>(s_code[i])[w];
            sum[i] = __dp4a(k.x, q.x, __dp4a(k.y, q.y, __dp4a(k.z, q.z, __dp4a(k.w, q.w, sum[i]))));
          }
        }
        int best = sums[j];
        for (int i = 0; i < heads; ++i) best = max(best, sum[i]);
        sums[j] = best;
      }
    }
    __syncthreads();
    for (int j = tid; j < n; j += kThreads) {
      const int page = table[j >> (c.page_log2 - bl)];
      uint32_t key = 0;
      if (unsigned(page) < unsigned(c.num_pages)) {
        key = kAlways;
        if (scored && j >= a.first && j < n - a.last) {
          const float s = a.i.scales[(int64_t(page) * c.kv_heads + h) * per_page + (j & (per_page - 1))];
          key = order_of(s < INFINITY ? float(sums[j]) * s : INFINITY);
        }
      }
      keys[j] = key;
    }
    __syncthreads();
    take_best(keys, n, a.count, out);
    __syncthreads();
  }
}

template <int G>
int launch_select(const PagedSelectArgs& a, cudaStream_t st) {
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  auto kern = paged_select_kernel<G>;
  e = once.run(dev, [&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SPECTRA_MAX_INDEXED_BLOCKS * 4);
  });
  if (e != cudaSuccess) return cuda_status(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.i.c.kv_heads), unsigned(std::min<int64_t>(a.i.c.total, 65535)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(a.max_blocks) * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a));
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
