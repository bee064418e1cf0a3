// Rotate-and-append and read-back of the paged INT4 KV cache for sm_100a.
//
// Append, for every new token at position p of its sequence: the pairs (a, b)
// of each query and key head are turned by the angle of p,
//   a' = a cos - b sin,  b' = b cos + a sin
// (halves of the rotated part, or neighbours), the queries are rounded once to
// their type, the keys stay in fp32 and go with the values, group of 32 by
// group, through
//   lo = min(0, x), hi = max(0, x), s = fp16((hi - lo) / 15), r = 1 / s
//   z = min(rint(-lo r), 15),  q = clamp(rint(x r) + z, 0, 15)
// into the cache; q stands for (q - z) s.  Zero is inside [lo, hi] by
// construction, so a group of one sign keeps its half step (the dense cache's
// quantiser, which repeats the reference's arithmetic, saturates there).  The
// codes are taken with the fp16-rounded scale that will be read back, and
// every operation is rounded by itself (no fma), so they can be reproduced
// bit for bit.  A group of the key or the value that holds a NaN or infinity,
// or spans more than 65472 (15 scales of more would pass fp16's largest
// number), has no code: its key group gets a NaN scale and its value group
// zeros, so exactly the rows that look at the token become NaN and value
// scales are always finite (a masked token's weight of 0 times its value is 0).
//
// One thread takes 8 features (16 bytes) of one head, four threads a group; where
// a query head is turned as a whole by halves, the pair of 8 that turn into each
// other, so that nothing is read twice.  A block takes 1 to 8 tokens; it looks up
// their sequences, positions and pages and brings their angles first.  With
// positions of several axes (time, height and width of a patch, say) pair i is
// turned by the row positions[axis of i][token] of the angles; they are loaded
// before the look-ups, so they add no load to the chain.  A row outside the
// table turns into NaN.
// Bound by HBM: 2 bytes in and out per query value, 2 in and 0.59 out per key
// or value.  Measured: append and read back of 16384 tokens, 64 query heads on
// 8, heads of 128, 162 us together (4.4 TB/s, 69 % of the copy rate), the same by three axes; one token
// of 128 sequences 20.7 us, which is the two calls on the host.
#include <math.h>

#include <algorithm>

#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

namespace {

constexpr int kThreads = 256;
constexpr float kMaxSpan = 65472.f;
constexpr int kTokens = kThreads / 32;  // tokens of a block, at most: a warp looks each of them up
constexpr int kAxes = 4;                // axes of a token's position, at most

template <bool BF16>
__device__ __forceinline__ float to_f(uint32_t bits16) {
  if constexpr (BF16) return __uint_as_float(bits16 << 16);
  return __half2float(__ushort_as_half(uint16_t(bits16)));
}
template <bool BF16>
__device__ __forceinline__ uint32_t from_f2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight values as they lie in memory, and as numbers.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const void* base, int64_t at) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = uint32_t(p[2 * i]) | (uint32_t(p[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <bool BF16>
__device__ __forceinline__ void numbers(const uint4& w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f<BF16>(v[i] & 0xFFFFu);
    x[2 * i + 1] = to_f<BF16>(v[i] >> 16);
  }
}

// The features of a thread, as loaded: eight, and those they are turned with
// (PAIR: its other eight; else the partners, where they are somewhere else).
struct Raw {
  uint4 own, other;
};
template <bool VEC, bool PAIR>
__device__ __forceinline__ Raw load_raw(const PagedAppendArgs& a, const void* base, int64_t at, int d) {
  Raw r;
  r.own = load8<VEC>(base, at + d);
  if constexpr (PAIR) {
    r.other = load8<VEC>(base, at + d + a.c.head_dim / 2);
  } else {
    const int half = a.rotary / 2;
    r.other = d < a.rotary && !a.interleaved ? load8<VEC>(base, at + (d >= half ? d - half : d + half)) : r.own;
  }
  return r;
}

// Turned by the angles in cs: cos of the rotary / 2 pairs, then sin.  PAIR: y the other eight.
template <bool BF16, bool PAIR>
__device__ __forceinline__ void turn(const PagedAppendArgs& a, const Raw& r, const float* cs, int d, float (&x)[8], float (&y)[8]) {
  numbers<BF16>(r.own, x);
  const int half = a.rotary / 2;
  if constexpr (PAIR) {
    numbers<BF16>(r.other, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = cs[d + i], s = cs[half + d + i], u = x[i], w = y[i];
      x[i] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
      y[i] = __fadd_rn(__fmul_rn(w, c), __fmul_rn(u, s));
    }
    return;
  }
  if (d >= a.rotary) return;
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = cs[d / 2 + i], s = cs[half + d / 2 + i], u = x[2 * i], w = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(w, c), __fmul_rn(u, s));
    }
    return;
  }
  const bool second = d >= half;
  const int i0 = second ? d - half : d;
  numbers<BF16>(r.other, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float own = __fmul_rn(x[i], cs[i0 + i]), other = __fmul_rn(y[i], cs[half + i0 + i]);
    x[i] = second ? __fadd_rn(own, other) : __fsub_rn(own, other);
  }
}

// Range of a group over its four threads, zero included; false where it has no codes.
__device__ __forceinline__ bool group_range(const float (&x)[8], unsigned quad, float& lo, float& hi) {
  lo = 0.f;
  hi = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = x[i] == x[i] ? fmaxf(hi, x[i]) : INFINITY;  // (min and max pass over a NaN)
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(quad, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(quad, hi, o));
  }
  return __fsub_rn(hi, lo) <= kMaxSpan;
}

// Codes of eight values, the first in the lowest nibble.
__device__ __forceinline__ uint32_t group_codes(const float (&x)[8], float lo, float hi, uint16_t& scale, uint8_t& zero) {
  const __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const float s32 = __half2float(s);
  const float r = s32 > 0.f ? __frcp_rn(s32) : 0.f;
  const float z = fminf(rintf(__fmul_rn(-lo, r)), 15.f);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf(rintf(__fmul_rn(x[i], r)) + z, 0.f), 15.f);
    w |= uint32_t(q) << (4 * i);
  }
  scale = __half_as_ushort(s);
  zero = uint8_t(z);
  return w;
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void store_q(const PagedAppendArgs& a, int64_t at, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = from_f2<BF16>(x[2 * i], x[2 * i + 1]);
  uint16_t* o = reinterpret_cast<uint16_t*>(a.q_out) + at;
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
  }
}

// Codes of the features d.. of a token into its tile; `quad`: the four threads of the group.
__device__ __forceinline__ void store_kv(const TileLayout L, uint8_t* tile, int pos, int d, unsigned quad, const float (&k)[8],
                                         const float (&v)[8]) {
  float klo, khi, vlo, vhi;
  bool ok = group_range(k, quad, klo, khi);
  ok = group_range(v, quad, vlo, vhi) && ok;
  uint32_t kw = 0, vw = 0;
  uint16_t ks = 0x7E00u, vs = 0;  // NaN and 0: what a group without codes gets
  uint8_t kz = 0, vz = 0;
  if (ok) {
    kw = group_codes(k, klo, khi, ks, kz);
    vw = group_codes(v, vlo, vhi, vs, vz);
  }
  const int g = d / 32, w = (d & 31) / 8, tok = pos & 15, row = tok & 7, pair = tok >> 1, odd = tok & 1;
  uint8_t* kc = tile + L.k_codes() + (tok >> 3) * L.block();
  uint8_t* vc = tile + L.v_codes() + (tok >> 3) * L.block();
  reinterpret_cast<uint32_t*>(kc)[(row * 4 + w) * L.G + g] = kw;
  uint16_t* vp = reinterpret_cast<uint16_t*>(vc) + odd;
  vp[2 * (((2 * w) * 4 + (row >> 1)) * L.G + g)] = uint16_t(vw);
  vp[2 * (((2 * w + 1) * 4 + (row >> 1)) * L.G + g)] = uint16_t(vw >> 16);
  if (w == 0) {
    reinterpret_cast<uint16_t*>(tile + L.k_scales())[tok * L.G + g] = ks;
    reinterpret_cast<uint16_t*>(tile + L.v_scales())[2 * (pair * L.G + g) + odd] = vs;
    tile[L.k_zeros() + tok * L.G + g] = kz;
    tile[L.v_zeros() + 2 * (pair * L.G + g) + odd] = vz;
  }
}

// Position (-1: padding) and tile of head 0 (NULL: no page) of a block's tokens, a warp each.
__device__ __forceinline__ void find_tokens(const PagedView& c, int64_t t0, int n, int* s_pos, uint8_t** s_tile) {
  const int i = threadIdx.x >> 5;
  if (i < n) {
    const int64_t t = t0 + i;
    const int b = sequence_of(c, t);
    int pos = -1;
    uint8_t* tile = nullptr;
    if (b >= 0) {
      int64_t first;
      int count;
      new_tokens(c, b, first, count);
      pos = c.seq_lens[b] - count + int(t - first);
      if (pos >= 0 && pos < c.limit)
        tile = tile_of(c, b, 0, pos);
      else
        pos = -1;
    }
    if ((threadIdx.x & 31) == 0) {
      s_pos[i] = pos;
      s_tile[i] = tile;
    }
  }
}

// (Five blocks an SM: many threads with one token's loads each in flight measured faster than few with
// several: 163 us against 169-198 for a prompt of 16384 with its read-back.)
// PAIR: a thread of the queries takes features d.. and d + D / 2.. (rotary = D, by halves).
template <bool BF16, bool VEC, bool PAIR>
__global__ void __launch_bounds__(kThreads, 5) paged_append_kernel(PagedAppendArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  extern __shared__ float s_angles[];  // [tokens][rotary]
  __shared__ int s_pos[kTokens];
  __shared__ uint8_t* s_tile[kTokens];
  __shared__ int s_axis[kAxes * kTokens];
  const PagedView& c = a.c;
  const int D = c.head_dim, half = D / 2;
  const int q_chunks = PAIR ? D / 16 : D / 8, kv_chunks = D / 8;
  const int q_items = a.q ? a.q_heads * q_chunks : 0;
  const int items = q_items + c.kv_heads * kv_chunks;
  const TileLayout L{D / 32};
  const int64_t head_bytes = int64_t(1 << (c.page_log2 - 4)) * L.bytes();
  const int item = blockIdx.x * kThreads + threadIdx.x;
  const bool is_q = item < q_items;
  const int of = is_q ? item : item - q_items, chunks = is_q ? q_chunks : kv_chunks;
  const int h = of / chunks, d = (of - h * chunks) * 8;
  // the four threads of a group are in step: q_items and kv_chunks are multiples of 4
  const unsigned quad = 0xFu << (threadIdx.x & 28);
  for (int64_t t0 = int64_t(blockIdx.y) * a.tokens; t0 < c.total; t0 += int64_t(gridDim.y) * a.tokens) {
    const int n = int(c.total - t0 < a.tokens ? c.total - t0 : a.tokens);
    if (a.positions && threadIdx.x < a.axes * kTokens) {
      const int axis = threadIdx.x / kTokens, i = threadIdx.x % kTokens;
      if (i < n) s_axis[threadIdx.x] = a.positions[axis * a.pos_rs + t0 + i];
    }
    find_tokens(c, t0, n, s_pos, s_tile);
    __syncthreads();
    const int turns = a.rotary / 2;
    for (int i = threadIdx.x; i < n * turns; i += kThreads) {
      const int k = i / turns, j = i - k * turns, pos = s_pos[k];
      if (pos >= 0) {
        int row = pos;  // (the host has checked that the table reaches every position)
        if (a.positions) row = s_axis[(a.pair_axes[j >> 4] >> (2 * (j & 15)) & 3) * kTokens + k];
        const bool in = row >= 0 && row < a.cs_rows;
        s_angles[k * a.rotary + j] = in ? a.cos[row * a.cs_rs + j] : NAN;
        s_angles[k * a.rotary + turns + j] = in ? a.sin[row * a.cs_rs + j] : NAN;
      }
    }
    __syncthreads();
    if (item < items) {
      if (is_q) {
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          float x[8], y[8];
          if (s_pos[i] >= 0) {
            const Raw raw = load_raw<VEC, PAIR>(a, a.q, (t0 + i) * a.q_ts + h * a.q_hs, d);
            turn<BF16, PAIR>(a, raw, s_angles + i * a.rotary, d, x, y);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
          }
          const int64_t at = (t0 + i) * a.qo_ts + h * a.qo_hs + d;
          store_q<BF16, VEC>(a, at, x);
          if constexpr (PAIR) store_q<BF16, VEC>(a, at + half, y);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          if (!s_tile[i]) continue;
          const int64_t t = t0 + i, at = t * a.v_ts + h * a.v_hs + d;
          const Raw raw = load_raw<VEC, false>(a, a.k, t * a.k_ts + h * a.k_hs, d);
          const uint4 v0 = load8<VEC>(a.v, at);
          float x[8], y[8], v[8];
          turn<BF16, false>(a, raw, s_angles + i * a.rotary, d, x, y);
          numbers<BF16>(v0, v);
          store_kv(L, s_tile[i] + h * head_bytes, s_pos[i], d, quad, x, v);
        }
      }
    }
    __syncthreads();
  }
}

// Eight features of one head of a token: (q - z) s, exact in fp32, rounded once.
__device__ __forceinline__ void store8(void* out, int64_t at, int dt, const float (&x)[8]) {
  if (dt == SPECTRA_DT_F32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = dt == SPECTRA_DT_BF16 ? from_f2<true>(x[2 * i], x[2 * i + 1]) : from_f2<false>(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(kThreads) paged_read_kernel(PagedReadArgs a) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  __shared__ uint8_t* s_tile[kTokens];
  __shared__ int s_pos[kTokens];
  constexpr int kAhead = 4;  // tokens whose loads are in flight
  const PagedView& c = a.c;
  const int chunks = c.head_dim / 8, items = c.kv_heads * chunks;
  const TileLayout L{c.head_dim / 32};
  const int64_t head_bytes = int64_t(1 << (c.page_log2 - 4)) * L.bytes();
  // few items: the block's threads take several tokens at once
  const int at_once = items < kThreads ? kThreads / items : 1;
  const int sub = items < kThreads ? threadIdx.x / items : 0;
  const int item = items < kThreads ? threadIdx.x - sub * items : blockIdx.x * kThreads + threadIdx.x;
  const int h = item / chunks, d = (item - h * chunks) * 8, g = d / 32, w = (d & 31) / 8;
  for (int64_t t0 = int64_t(blockIdx.y) * a.tokens; t0 < c.total; t0 += int64_t(gridDim.y) * a.tokens) {
    const int n = int(c.total - t0 < a.tokens ? c.total - t0 : a.tokens);
    find_tokens(c, t0, n, s_pos, s_tile);
    __syncthreads();
    if (item < items && sub < at_once) {
      for (int i0 = sub; i0 < n; i0 += kAhead * at_once) {
        uint32_t kw[kAhead], vw[kAhead], s2[kAhead], z2[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * at_once;
          kw[u] = vw[u] = s2[u] = z2[u] = 0;
          if (i < n && s_tile[i]) {
            const uint8_t* tile = s_tile[i] + h * head_bytes;
            const int tok = s_pos[i] & 15, row = tok & 7, pair = tok >> 1, odd = tok & 1;
            const uint8_t* kc = tile + L.k_codes() + (tok >> 3) * L.block();
            const uint16_t* vp = reinterpret_cast<const uint16_t*>(tile + L.v_codes() + (tok >> 3) * L.block()) + odd;
            kw[u] = reinterpret_cast<const uint32_t*>(kc)[(row * 4 + w) * L.G + g];
            vw[u] = uint32_t(vp[2 * (((2 * w) * 4 + (row >> 1)) * L.G + g)]) |
                    (uint32_t(vp[2 * (((2 * w + 1) * 4 + (row >> 1)) * L.G + g)]) << 16);
            s2[u] = uint32_t(reinterpret_cast<const uint16_t*>(tile + L.k_scales())[tok * L.G + g]) |
                    (uint32_t(reinterpret_cast<const uint16_t*>(tile + L.v_scales())[2 * (pair * L.G + g) + odd]) << 16);
            z2[u] = uint32_t(tile[L.k_zeros() + tok * L.G + g]) | (uint32_t(tile[L.v_zeros() + 2 * (pair * L.G + g) + odd]) << 16);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * at_once;
          if (i >= n) break;
          const float ks = to_f<false>(s2[u] & 0xFFFFu), vs = to_f<false>(s2[u] >> 16);
          const float kz = float(z2[u] & 0xFFu), vz = float(z2[u] >> 16);
          float k[8], v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            k[j] = __fmul_rn(float((kw[u] >> (4 * j)) & 15u) - kz, ks);
            v[j] = __fmul_rn(float((vw[u] >> (4 * j)) & 15u) - vz, vs);
          }
          const int64_t at = ((t0 + i) * c.kv_heads + h) * c.head_dim + d;
          store8(a.k, at, a.out_dtype, k);
          store8(a.v, at, a.out_dtype, v);
        }
      }
    }
    __syncthreads();
  }
}

// Tokens of a block: as many as leave some blocks for every SM.
int block_tokens(int64_t total, int64_t item_blocks, int sms) {
  int n = kTokens;
  while (n > 1 && total * item_blocks < int64_t(n) * sms * 8) n /= 2;
  return n;
}

template <class Args>
int launch(void (*kernel)(Args), Args a, int items, int angles, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  const int item_blocks = (items + kThreads - 1) / kThreads;
  a.tokens = block_tokens(a.c.total, item_blocks, device_sms(dev));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(item_blocks), unsigned(std::min<int64_t>((a.c.total + a.tokens - 1) / a.tokens, 65535)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(a.tokens) * angles * sizeof(float);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a));
}

template <bool BF16>
int launch_append(const PagedAppendArgs& a, bool pair, int items, cudaStream_t st) {
  if (pair) return launch(a.vec ? paged_append_kernel<BF16, true, true> : paged_append_kernel<BF16, false, true>, a, items, a.rotary, st);
  return launch(a.vec ? paged_append_kernel<BF16, true, false> : paged_append_kernel<BF16, false, false>, a, items, a.rotary, st);
}

}  // namespace

int launch_paged_append(const PagedAppendArgs& a, cudaStream_t st) {
  // the whole head turned, by halves of whole 16-byte pieces; a multiple of 4 of them keeps groups in step
  const bool pair = a.rotary == a.c.head_dim && !a.interleaved && a.c.head_dim % 64 == 0;
  const int items = a.q_heads * (a.c.head_dim / (pair ? 16 : 8)) + a.c.kv_heads * (a.c.head_dim / 8);
  return a.dtype == SPECTRA_DT_BF16 ? launch_append<true>(a, pair, items, st) : launch_append<false>(a, pair, items, st);
}

int launch_paged_read(const PagedReadArgs& a, cudaStream_t st) {
  return launch(paged_read_kernel, a, a.c.kv_heads * (a.c.head_dim / 8), 0, st);
}

}  // namespace spectra
