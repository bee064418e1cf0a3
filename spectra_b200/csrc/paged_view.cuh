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

// The same with the attention's rows: only the first max_q tokens have any; `extra` is how many have none.
__device__ __forceinline__ void new_rows(const PagedView& c, int b, int64_t& first, int& count, int& extra) {
  new_tokens(c, b, first, count);
  extra = count > c.max_q ? count - c.max_q : 0;
  count -= extra;
}

// Sequence of new token t, or -1 where none holds it; the whole warp asks for one
// token.  (A 32-way search: two loads that wait for each other up to 1024 sequences.)
__device__ __forceinline__ int sequence_of(const PagedView& c, int64_t t) {
  if (!c.cu_q) {
    const int64_t b = t / c.q_len;
    return b < c.batch ? int(b) : -1;
  }
  const int lane = threadIdx.x & 31;
  int at = -1, step = c.batch + 1;  // cu_q[at] <= t (or at = -1) < cu_q[at + step + 1]
  while (step > 1) {
    step = (step + 31) / 32;
    const int64_t i = int64_t(at) + int64_t(lane + 1) * step;
    const bool below = i <= c.batch && c.cu_q[i] <= t;
    at += __popc(__ballot_sync(0xffffffffu, below)) * step;
  }
  return at >= 0 && at < c.batch ? at : -1;
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

// First key that a row at `pos` may see (window 0: none; pos negative: padding).  Any window up to
// INT32_MAX: nothing is computed that 32 bits do not hold.
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// Scores are kept in powers of two.  A running maximum is raised when a score
// passes it by more than kLazy.
constexpr float kLazy = 8.f;
// Weights are kept times 2^kShift (their sums too, so nothing else changes): the
// smallest that fp16 holds as normal numbers lie 2^-17 below the maximum's, and
// above it fp16 has 12 bits for scores that pass a maximum that was not raised.
// (More would raise it more often: prompts with a cap, heads of 64, took 417 us
// with 5, 408 with 3, 401 with 1.)
constexpr float kShift = 3.f;
constexpr float kNone = -3e38f;  // below every score that is seen, as far as fp32 holds scores
// A weight's exponent is one fma of the product, its factor and the maximum.  That leaves what the
// maximum was rounded by, a share 2^-24 of it: under kLoud less than 2^-4 and the same for every key,
// above it the product is rounded first (a maximum near 2^31 would give exponents past fp32's).
constexpr float kLoud = 1048576.f;
constexpr float kLog2e = 1.4426950408889634f;

// BYTES of shared memory into registers, as wide as their alignment allows.
template <int BYTES>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[(BYTES + 3) / 4]) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 8; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(p)[i];
      w[2 * i] = v.x; w[2 * i + 1] = v.y;
    }
  } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else if constexpr (BYTES % 2 == 0) {
#pragma unroll
    for (int i = 0; i < (BYTES + 3) / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < BYTES / 2; ++i) w[i >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  } else {
#pragma unroll
    for (int i = 0; i < (BYTES + 3) / 4; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < BYTES; ++i) w[i >> 2] |= uint32_t(p[i]) << (8 * (i & 3));
  }
}

// fp16's 1024.0 twice, as a register: with the mask as the immediate, mask-and-or
// is one instruction (two constants would make it two).
__device__ __forceinline__ uint32_t fp16_1024() {
  uint32_t r;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(r));
  return r;
}
// 1024 + q of bits 0-3 of both halves; 1024 + 16 q of bits 4-7.
__device__ __forceinline__ uint32_t code_low(uint32_t w, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(magic));
  return r;
}
__device__ __forceinline__ uint32_t code_high(uint32_t w, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r) : "r"(w), "r"(magic));
  return r;
}

__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_pack(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return hi ? __high2float(h) : __low2float(h);
}
// 1024 + byte, of bytes 2 i and 2 i + 1 of w.
__device__ __forceinline__ uint32_t byte_pair(uint32_t w, int i) {
  return __byte_perm(w, 0x64646464u, i ? 0x4342u : 0x4140u);
}
// D = A B + C of mma.sync m16n8k16, fp16 in, fp32 out.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, const float4& c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// tanh(x) = x P(x^2), on the FMA pipe where tanh_exp takes two of the special-function
// unit's turns: fits of tanh(x) / x in powers of x^2 with P(0) = 1, for the least maximum
// of the relative error (own computation: iteratively reweighted least squares on Chebyshev
// nodes), so that a score is off by a share of itself whatever its cap.  Six terms for
// |x| <= 0.95 (prompts' usual steps), error 4.1e-7 (4.9e-7 with fp32's roundings); four for
// |x| <= 0.5 (high_cap), 6.5e-7 (7.2e-7).
constexpr float kTanhRange6 = 0.95f * 0.95f, kTanhRange4 = 0.5f * 0.5f;
__device__ constexpr float kTanhFit6[6] = {1.f, -0.3333132863044739f, 0.13300810754299164f, -0.05221107602119446f,
                                           0.017525605857372284f, -0.003422057954594493f};
__device__ constexpr float kTanhFit4[4] = {1.f, -0.33328160643577576f, 0.13205359876155853f, -0.0447506383061409f};
// Larger magnitude of both halves (bf16 or fp16; a NaN is passed over), as bits.
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  b &= 0x7FFF7FFFu;
  if constexpr (BF16) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// tanh by its exponential: absolute error up to 2^-21 over the whole range, so not for small |x|.
__device__ __forceinline__ float tanh_exp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(2.f * kLog2e * x)));
  return fmaf(-2.f, r, 1.f);
}
// A product's factor for the cap's argument; finite, so that 0 stays 0 under the smallest caps.
__device__ __forceinline__ float cap_factor(float factor, float cap) { return fminf(factor / cap, 1e37f); }
// Up to this cap tanh_exp's absolute error is less than 2^-14 of a score (in powers of e), and serves as
// it is (high_cap in its place cost 40 us of the 450 that capped prompts took).
constexpr float kLowCap = 128.f;
// Under a higher one: the product that, uncapped, has the capped score of v, to 2^-20 of itself.
// back = 1 / inv (an infinity where inv vanishes, which is not used: then x does too).
__device__ __forceinline__ float high_cap(float v, float inv, float back) {
  const float x = v * inv, u = x * x;
  float r = kTanhFit4[3];
#pragma unroll
  for (int d = 2; d >= 0; --d) r = fmaf(r, u, kTanhFit4[d]);
  return u <= kTanhRange4 ? v * r : tanh_exp(x) * back;
}

}  // namespace spectra
