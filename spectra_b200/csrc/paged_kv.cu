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
// or spans more than 65472 (15 scales of more would pass fp16's largest number), has no code: its key group gets a NaN scale and
// its value group zeros, so exactly the rows that look at the token become
// NaN and value scales are always finite (a masked token's weight of 0 times
// its value is 0).
//
// One thread takes 8 features (16 bytes) of one head, four threads a group.
// Bound by HBM: 2 bytes in and out per query value, 2 in and 0.59 out per key
// or value.
#include <math.h>

#include <algorithm>

#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

namespace {

constexpr int kThreads = 256;
constexpr float kMaxSpan = 65472.f;

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

template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + at;
  if constexpr (VEC) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = to_f<BF16>(v[i] & 0xFFFFu);
      x[2 * i + 1] = to_f<BF16>(v[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f<BF16>(p[i]);
  }
}

// Eight features d.. of a head at `at`, turned by the position's angles.
template <bool BF16, bool VEC>
__device__ __forceinline__ void load_rotated(const PagedAppendArgs& a, const void* base, int64_t at, int d, int pos,
                                             float (&x)[8]) {
  load8<BF16, VEC>(base, at + d, x);
  if (d >= a.rotary) return;
  const float* cs = a.cos + pos * a.cs_rs;
  const float* sn = a.sin + pos * a.cs_rs;
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = cs[d / 2 + i], s = sn[d / 2 + i], u = x[2 * i], w = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(w, c), __fmul_rn(u, s));
    }
    return;
  }
  const int half = a.rotary / 2;
  const bool second = d >= half;
  const int i0 = second ? d - half : d;
  float y[8];
  load8<BF16, VEC>(base, at + (second ? d - half : d + half), y);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = cs[i0 + i], s = sn[i0 + i];
    const float own = __fmul_rn(x[i], c), other = __fmul_rn(y[i], s);
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
__global__ void __launch_bounds__(kThreads) paged_append_kernel(PagedAppendArgs a) {
  sm100::pdl_wait();
  const PagedView& c = a.c;
  const int chunks = c.head_dim / 8;
  const int q_items = a.q ? a.q_heads * chunks : 0;
  const int items = q_items + c.kv_heads * chunks;
  const TileLayout L{c.head_dim / 32};
  const int item = blockIdx.x * kThreads + threadIdx.x;
  for (int64_t t = blockIdx.y; t < c.total; t += gridDim.y) {
    const int b = sequence_of(c, t);
    int pos = -1;
    if (b >= 0) {
      int64_t first;
      int count;
      new_tokens(c, b, first, count);
      pos = c.seq_lens[b] - count + int(t - first);
    }
    const bool real = pos >= 0 && pos < c.limit;
    if (item < q_items) {
      const int h = item / chunks, d = (item - h * chunks) * 8;
      float x[8];
      if (real) {
        load_rotated<BF16, VEC>(a, a.q, t * a.q_ts + h * a.q_hs, d, pos, x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
      }
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = from_f2<BF16>(x[2 * i], x[2 * i + 1]);
      uint16_t* o = reinterpret_cast<uint16_t*>(a.q_out) + t * a.qo_ts + h * a.qo_hs + d;
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
      }
    } else if (item < items && real) {
      const int kv = item - q_items;
      const int h = kv / chunks, d = (kv - h * chunks) * 8;
      // the four threads of a group are in step: q_items and chunks are multiples of 4
      const unsigned quad = 0xFu << (threadIdx.x & 28);
      float k[8], v[8], klo, khi, vlo, vhi;
      load_rotated<BF16, VEC>(a, a.k, t * a.k_ts + h * a.k_hs, d, pos, k);
      load8<BF16, VEC>(a.v, t * a.v_ts + h * a.v_hs + d, v);
      uint8_t* tile = tile_of(c, b, h, pos);
      bool ok = group_range(k, quad, klo, khi);
      ok = group_range(v, quad, vlo, vhi) && ok;
      uint32_t kw = 0, vw = 0;
      uint16_t ks = 0x7E00u, vs = 0;  // NaN and 0: what a group without codes gets
      uint8_t kz = 0, vz = 0;
      if (ok) {
        kw = group_codes(k, klo, khi, ks, kz);
        vw = group_codes(v, vlo, vhi, vs, vz);
      }
      if (tile) {
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
    }
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
  const PagedView& c = a.c;
  const int chunks = c.head_dim / 8, items = c.kv_heads * chunks;
  const TileLayout L{c.head_dim / 32};
  const int item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= items) return;
  const int h = item / chunks, d = (item - h * chunks) * 8, g = d / 32, w = (d & 31) / 8;
  for (int64_t t = blockIdx.y; t < c.total; t += gridDim.y) {
    const int b = sequence_of(c, t);
    int pos = -1;
    if (b >= 0) {
      int64_t first;
      int count;
      new_tokens(c, b, first, count);
      pos = c.seq_lens[b] - count + int(t - first);
    }
    const uint8_t* tile = pos >= 0 && pos < c.limit ? tile_of(c, b, h, pos) : nullptr;
    float k[8] = {}, v[8] = {};
    if (tile) {
      const int tok = pos & 15, row = tok & 7, pair = tok >> 1, odd = tok & 1;
      const uint8_t* kc = tile + L.k_codes() + (tok >> 3) * L.block();
      const uint8_t* vc = tile + L.v_codes() + (tok >> 3) * L.block();
      const uint32_t kw = reinterpret_cast<const uint32_t*>(kc)[(row * 4 + w) * L.G + g];
      const uint16_t* vp = reinterpret_cast<const uint16_t*>(vc) + odd;
      const uint32_t vw = uint32_t(vp[2 * (((2 * w) * 4 + (row >> 1)) * L.G + g)]) |
                          (uint32_t(vp[2 * (((2 * w + 1) * 4 + (row >> 1)) * L.G + g)]) << 16);
      const float ks = to_f<false>(reinterpret_cast<const uint16_t*>(tile + L.k_scales())[tok * L.G + g]);
      const float vs = to_f<false>(reinterpret_cast<const uint16_t*>(tile + L.v_scales())[2 * (pair * L.G + g) + odd]);
      const float kz = float(tile[L.k_zeros() + tok * L.G + g]);
      const float vz = float(tile[L.v_zeros() + 2 * (pair * L.G + g) + odd]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        k[i] = __fmul_rn(float((kw >> (4 * i)) & 15u) - kz, ks);
        v[i] = __fmul_rn(float((vw >> (4 * i)) & 15u) - vz, vs);
      }
    }
    const int64_t at = (t * c.kv_heads + h) * c.head_dim + d;
    store8(a.k, at, a.out_dtype, k);
    store8(a.v, at, a.out_dtype, v);
  }
}

template <class Args>
int launch(void (*kernel)(Args), const Args& a, int items, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((items + kThreads - 1) / kThreads), unsigned(std::min<int64_t>(a.c.total, 65535)));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a));
}

}  // namespace

int launch_paged_append(const PagedAppendArgs& a, cudaStream_t st) {
  const int items = ((a.q ? a.q_heads : 0) + a.c.kv_heads) * (a.c.head_dim / 8);
  if (a.dtype == SPECTRA_DT_BF16)
    return launch(a.vec ? paged_append_kernel<true, true> : paged_append_kernel<true, false>, a, items, st);
  return launch(a.vec ? paged_append_kernel<false, true> : paged_append_kernel<false, false>, a, items, st);
}

int launch_paged_read(const PagedReadArgs& a, cudaStream_t st) {
  return launch(paged_read_kernel, a, a.c.kv_heads * (a.c.head_dim / 8), st);
}

}  // namespace spectra
