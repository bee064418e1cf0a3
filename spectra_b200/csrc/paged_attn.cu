// Attention over the paged INT4 KV cache for sm_100a: one or a few new tokens
// per sequence.
//
// Row (token i at position p, query head h) over the keys n it sees:
//   t_n = scale * q . k_n;  t = cap tanh(t / cap);  t += slope_h (n - p)
//   o = sum_n e^(t_n - m) v_n / sum_n e^(t_n - m)
// with a running maximum m, in one pass over the cache: every byte of it is
// read once per row tile.  Rows of one key/value head (its `group` query
// heads times the new tokens) are the columns of the tensor-core products, so
// the codes are unpacked once for all of them.
//
// Products (mma.sync m16n8k16, fp32 accumulation; with 1-16 rows per head the
// tcgen05 shapes would be mostly padding, and the kernel is bound by bytes
// and by unpacking instructions, not by the tensor pipe):
//   S^T = K Q^T: A = raw key codes offset + q (128 + q in bf16, 1024 + q in
//     fp16: one mask-and-or per pair), 16 tokens x 16 features; per group of
//     32 features the accumulator starts at -offset * X, X = sum of q over the
//     group, and t = s (D - z X) in fp32: the keys are never rounded.
//   O^T = V^T P^T: A = values (q - z) s in fp16 (exact difference, one
//     rounding of the product, 11 bits), B = P in fp16, transposed in
//     registers (movmatrix).  P <= 2^kLazy, so fp16 holds it; its rounding
//     (2^-12) averages over the keys.
// The running maximum is only raised when a score passes it by more than
// kLazy (in powers of two): most tiles need no cross-lane reduction and no
// rescaling of O.
//
// Work: a segment is (sequence, key/value head, row tile); a unit is 32
// consecutive tokens of a segment.  The units of all segments, laid end to
// end, are dealt to the CTAs in equal contiguous shares, whatever the lengths
// of the sequences; a segment that several CTAs share is put together by the
// last of them to finish, always in the same order.
#include <math.h>

#include <algorithm>

#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

__device__ int g_paged_attn_timeouts = 0;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnit = 32;          // tokens of a unit: two tiles
constexpr int kStages = 2;         // units in flight per warp
constexpr int kMaxCtas = int(kPagedCounterBytes / sizeof(int));

struct AttnParams {
  PagedAttnArgs a;
  int* counters;
  float* partials;
  int min_share;                   // units a CTA takes at least
  int max_rows;                    // a sequence with more rows per head is the other kernel's
};

// ------------------------------------------------------------ the batch
struct Span {  // a sequence's rows and the keys its rows look at
  int64_t first;  // first new token
  int count;      // new tokens
  int len;        // keys (cut to the batch's limit)
  int pos0;       // position of the first new token
  int unit0;      // first unit that any row looks at
  int units;      // units of one segment, at least 1
  int tiles;      // row tiles
};

template <int ROWS>
__device__ __forceinline__ Span span_of(const AttnParams& p, int b) {
  const PagedAttnArgs& a = p.a;
  Span s;
  new_tokens(a.c, b, s.first, s.count);
  const int len = a.c.seq_lens[b];
  s.pos0 = len - s.count;
  s.len = len < 0 ? 0 : (len < a.c.limit ? len : a.c.limit);
  s.tiles = s.count * a.group > p.max_rows ? 0 : (s.count * a.group + ROWS - 1) / ROWS;
  const int lo = a.window > 0 ? max(0, s.pos0 - a.window + 1) : 0;
  s.unit0 = lo / kUnit;
  s.units = max(1, (s.len + kUnit - 1) / kUnit - s.unit0);
  return s;
}

template <int G, int NT>
struct Cfg {
  static constexpr int D = 32 * G;
  static constexpr int ROWS = 8 * NT;
  static constexpr int kTile = TileLayout{G}.bytes();
  static constexpr int kStage = 2 * kTile;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kSlab = ROWS * (D + 4);               // one warp's partial result, floats
  static constexpr int kMerge = kWarps * kSlab * 4;           // shares the ring's memory
  static constexpr int kBig = kRing > kMerge ? kRing : kMerge;
  static constexpr int kQ = G * NT * 32 * 16;                 // query fragments
  static constexpr int kX = G * NT * 4 * 16;                  // {-offset X, X} of a lane's two rows
  static constexpr int kMeta = ROWS * 16;                     // hi, lo, slope, position of a row
  static constexpr int kSmem = kBig + kQ + kX + kMeta + kWarps * kStages * 8 + 64;
  static constexpr int kPartial = ROWS * (D + 2);             // floats of one CTA's partial result
};

// ------------------------------------------------------------ the kernel
template <bool BF16, int G, int NT, bool MOD>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(AttnParams p) {
  using C = Cfg<G, NT>;
  constexpr int D = C::D, ROWS = C::ROWS;
  constexpr uint32_t kKeyMagic = BF16 ? 0x43004300u : 0x64006400u;
  constexpr float kKeyOffset = BF16 ? 128.f : 1024.f;
  constexpr TileLayout L{G};
  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;

  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem);
  uint4* qfrag = reinterpret_cast<uint4*>(smem + C::kBig);
  float4* xs = reinterpret_cast<float4*>(smem + C::kBig + C::kQ);
  int4* meta = reinterpret_cast<int4*>(smem + C::kBig + C::kQ + C::kX);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBig + C::kQ + C::kX + C::kMeta);
  __shared__ long long s_scan[kWarps];
  __shared__ long long s_base;
  __shared__ int s_seq, s_last;
  __shared__ volatile int s_stop;     // a copy did not arrive: no further ones
  __shared__ int s_held[kWarps * kStages];  // tiles of a stage that a page holds
  __shared__ volatile int s_never;    // 0: each warp waits for its own copies, whatever the others saw

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
  if (tid < kWarps * kStages) sm100::mbar_init(bars + tid, 1);
  if (tid == 0) {
    s_stop = s_never = 0;
    s_seq = -1;
  }
  sm100::fence_mbar_init();
  __syncthreads();
  sm100::pdl_wait();

  // ---- this CTA's share of the units
  long long total = 0;
  for (int b0 = 0; b0 < c.batch; b0 += kThreads) {
    if (b0 + tid < c.batch) {
      const Span s = span_of<ROWS>(p, b0 + tid);
      total += (long long)(s.units) * s.tiles * c.kv_heads;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_scan[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += s_scan[w];
  long long share = (total + gridDim.x - 1) / gridDim.x;
  if (share < p.min_share) share = p.min_share;
  const long long begin = share * blockIdx.x;
  const long long end = begin + share < total ? begin + share : total;

  // rows that belong to no sequence
  if (c.cu_q) {
    const int held = c.cu_q[c.batch];
    const int64_t row_words = int64_t(a.q_heads) * D;
    for (int64_t t = (held < 0 ? 0 : held) + int64_t(blockIdx.x); t < c.total; t += gridDim.x)
      for (int64_t i = tid; i < row_words; i += kThreads)
        reinterpret_cast<uint16_t*>(a.out)[t * a.o_ts + (i / D) * a.o_hs + i % D] = 0;
  }
  if (begin >= end) return;

  // ---- the sequence where the share begins
  long long base = 0;
  for (int b0 = 0; b0 < c.batch; b0 += kThreads) {
    long long mine = 0;
    if (b0 + tid < c.batch) {
      const Span s = span_of<ROWS>(p, b0 + tid);
      mine = (long long)(s.units) * s.tiles * c.kv_heads;
    }
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    long long before = base + sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      all += s_scan[w];
    }
    if (before <= begin && begin < before + mine) {
      s_seq = b0 + tid;
      s_base = before;
    }
    base += all;
    if (base > begin) break;
  }
  __syncthreads();
  int b = s_seq;
  long long seq_base = s_base;
  if (b < 0) return;

  const float c_exp = MOD ? 1.f : a.scale * kLog2e;
  uint32_t phase = 0;  // a bit for each stage
  long long at = begin;

  while (at < end) {
    // ---- the segment that holds unit `at`
    Span s = span_of<ROWS>(p, b);
    long long seq_units = (long long)(s.units) * s.tiles * c.kv_heads;
    while (at >= seq_base + seq_units) {
      seq_base += seq_units;
      ++b;
      s = span_of<ROWS>(p, b);
      seq_units = (long long)(s.units) * s.tiles * c.kv_heads;
    }
    const int seg = int((at - seq_base) / s.units);
    const long long seg_begin = seq_base + (long long)(seg) * s.units, seg_end = seg_begin + s.units;
    const int head = seg / s.tiles, row0 = (seg - head * s.tiles) * ROWS;
    const int u_begin = s.unit0 + int(at - seg_begin);
    const int u_end = s.unit0 + int((seg_end < end ? seg_end : end) - seg_begin);
    const int rows = min(ROWS, s.count * a.group - row0);

    // ---- units to load: warp w takes u_begin + w, + kWarps, ...
    auto issue = [&](int u, int stage) {
      if (lane < 2) {
        const int pos = u * kUnit + lane * kTileTokens;
        const uint8_t* src = pos < s.len ? tile_of(c, b, head, pos) : nullptr;
        uint64_t* bar = bars + warp * kStages + stage;
        uint8_t* dst = ring + (warp * kStages + stage) * C::kStage + lane * C::kTile;
        const unsigned held = __ballot_sync(0x3u, src != nullptr);
        if (lane == 0) {
          s_held[warp * kStages + stage] = int(held);
          sm100::mbar_arrive_expect_tx(bar, __popc(held) * C::kTile);
        }
        __syncwarp(0x3u);
        if (src) {
          bulk_g2s(dst, src, C::kTile, bar);
        } else {  // its keys are masked; its values have to be finite
          for (int i = L.v_codes(); i < C::kTile; i += 4) *reinterpret_cast<uint32_t*>(dst + i) = 0;
          sm100::fence_proxy_async_smem();
        }
      }
    };
    int next = u_begin + warp;
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      if (next + st * kWarps < u_end) issue(next + st * kWarps, st);
    }

    // ---- query fragments: X and the two products' B registers
    for (int i = tid; i < G * NT * 32; i += kThreads) {
      const int grp = i / (NT * 32), nt = (i / 32) % NT, row = row0 + nt * 8 + g;
      float x[8] = {};
      uint32_t raw[4] = {};
      if (nt * 8 + g < rows) {
        const int tok = row / a.group, h = head * a.group + row - tok * a.group;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (s.first + tok) * a.q_ts + h * a.q_hs + grp * 32 + cc * 8;
        if (a.vec) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) raw[j >> 1] |= uint32_t(src[j]) << (16 * (j & 1));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t bits = (raw[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
          x[j] = BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(uint16_t(bits)));
        }
      }
      // pairs (0,4) (1,5) (2,6) (3,7): the order in which the code pairs come
      qfrag[i] = make_uint4(__byte_perm(raw[0], raw[2], 0x5410), __byte_perm(raw[0], raw[2], 0x7632),
                            __byte_perm(raw[1], raw[3], 0x5410), __byte_perm(raw[1], raw[3], 0x7632));
      float sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float other = __shfl_xor_sync(0xffffffffu, sum, 4);  // row g ^ 1
      if (cc == 0 && (g & 1) == 0)
        xs[(grp * NT + nt) * 4 + g / 2] = make_float4(-kKeyOffset * sum, -kKeyOffset * other, sum, other);
    }
    if (tid < ROWS) {
      int hi = 0, lo = 0, pos = 0;
      float slope = 0.f;
      if (tid < rows) {
        const int tok = (row0 + tid) / a.group, h = head * a.group + (row0 + tid) - tok * a.group;
        pos = s.pos0 + tok;
        if (pos >= 0) hi = a.causal ? min(s.len, pos + 1) : s.len;
        if (a.window > 0) lo = max(0, pos - a.window + 1);
        if (a.slopes) slope = a.slopes[h] * kLog2e;
      }
      meta[tid] = make_int4(hi, lo, __float_as_int(slope), pos);
    }
    __syncthreads();
    // keys that every row sees: no mask needed
    int all_hi = 0x7FFFFFFF, all_lo = 0;
    for (int r = 0; r < rows; ++r) {
      all_hi = min(all_hi, meta[r].x);
      all_lo = max(all_lo, meta[r].y);
    }

    float o[G][2][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kNone;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < G * 2 * 4; ++i) o[i / 8][(i / 4) & 1][nt][i & 3] = 0.f;
    }

    int stage = 0;
    for (int u = next; u < u_end; u += kWarps) {
      if (!sm100::mbar_wait(bars + warp * kStages + stage, (phase >> stage) & 1u, &s_never)) {
        s_stop = 1;
        if (lane == 0) atomicAdd(&g_paged_attn_timeouts, 1);
      }
      const int held = s_held[warp * kStages + stage];
      const uint8_t* buf = ring + (warp * kStages + stage) * C::kStage;

      // ---- scores of 32 tokens: s[tile][nt][4], tokens g, g + 8, rows 2cc, 2cc + 1
      float sc[2][NT][4];
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const uint8_t* t = buf + tile * C::kTile;
        uint32_t w0[G], w1[G], ks0[(2 * G + 3) / 4], ks1[(2 * G + 3) / 4], kz0[(G + 3) / 4], kz1[(G + 3) / 4];
        lds<4 * G>(t + L.k_codes() + lane * 4 * G, w0);
        lds<4 * G>(t + L.k_codes() + L.block() + lane * 4 * G, w1);
        lds<2 * G>(t + L.k_scales() + g * 2 * G, ks0);
        lds<2 * G>(t + L.k_scales() + (g + 8) * 2 * G, ks1);
        lds<G>(t + L.k_zeros() + g * G, kz0);
        lds<G>(t + L.k_zeros() + (g + 8) * G, kz1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[tile][nt][i] = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          const uint32_t a0 = code_pair<0>(w0[grp], kKeyMagic), a1 = code_pair<0>(w1[grp], kKeyMagic);
          const uint32_t a2 = code_pair<1>(w0[grp], kKeyMagic), a3 = code_pair<1>(w1[grp], kKeyMagic);
          const uint32_t a4 = code_pair<2>(w0[grp], kKeyMagic), a5 = code_pair<2>(w1[grp], kKeyMagic);
          const uint32_t a6 = code_pair<3>(w0[grp], kKeyMagic), a7 = code_pair<3>(w1[grp], kKeyMagic);
          const float s0 = half_of(ks0[grp >> 1], grp & 1), s1 = half_of(ks1[grp >> 1], grp & 1);
          const float z0 = byte_of(kz0[grp >> 2], grp & 3), z1 = byte_of(kz1[grp >> 2], grp & 3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 q = qfrag[(grp * NT + nt) * 32 + lane];
            const float4 x = xs[(grp * NT + nt) * 4 + cc];
            float d[4] = {x.x, x.y, x.x, x.y};
            mma16816<BF16>(d, a0, a1, a2, a3, q.x, q.y);
            mma16816<BF16>(d, a4, a5, a6, a7, q.z, q.w);
            sc[tile][nt][0] = fmaf(s0, fmaf(-z0, x.z, d[0]), sc[tile][nt][0]);
            sc[tile][nt][1] = fmaf(s0, fmaf(-z0, x.w, d[1]), sc[tile][nt][1]);
            sc[tile][nt][2] = fmaf(s1, fmaf(-z1, x.z, d[2]), sc[tile][nt][2]);
            sc[tile][nt][3] = fmaf(s1, fmaf(-z1, x.w, d[3]), sc[tile][nt][3]);
          }
        }
      }

      // ---- cap, bias, mask
      const int n0 = u * kUnit;
      if constexpr (MOD) {
        const float inv = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int4 r = meta[nt * 8 + 2 * cc + j];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float& v = sc[k >> 1][nt][2 * (k & 1) + j];
              const float t = a.softcap > 0.f ? a.softcap * tanh_exp(v * inv) : v * a.scale;
              v = fmaf(__int_as_float(r.z), float(n0 + 8 * k + g - r.w), t * kLog2e);
            }
          }
      }
      if (n0 < all_lo || n0 + kUnit > all_hi || held != 3) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int4 r = meta[nt * 8 + 2 * cc + j];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int n = n0 + 8 * k + g;
              if (n >= r.x || n < r.y || !((held >> (k >> 1)) & 1u)) sc[k >> 1][nt][2 * (k & 1) + j] = -INFINITY;
            }
          }
      }

      // ---- running maximum, weights
      bool raise = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = fmaxf(fmaxf(sc[0][nt][j], sc[0][nt][2 + j]), fmaxf(sc[1][nt][j], sc[1][nt][2 + j])) * c_exp;
          raise = raise || top[nt][j] > m[nt][j] + kLazy;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float t = top[nt][j];
#pragma unroll
            for (int k = 4; k <= 16; k <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, k));
            t = fmaxf(t, m[nt][j]);
            const float f = exp2f(m[nt][j] - t);
            m[nt][j] = t;
            l[nt][j] *= f;
#pragma unroll
            for (int grp = 0; grp < G; ++grp)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                o[grp][h][nt][j] *= f;
                o[grp][h][nt][2 + j] *= f;
              }
          }
      }
      uint32_t pb[2][NT][2];  // P^T fragments: rows as columns
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"(fmaf(sc[tile][nt][i], c_exp, -m[nt][i & 1])));
            l[nt][i & 1] += e[i];
          }
          pb[tile][nt][0] = transpose8x8(h2_pack(e[0], e[1]));
          pb[tile][nt][1] = transpose8x8(h2_pack(e[2], e[3]));
        }

      // ---- values
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const uint8_t* t = buf + tile * C::kTile;
        uint32_t w0[G], w1[G], vs0[G], vs1[G], vz0[(2 * G + 3) / 4], vz1[(2 * G + 3) / 4];
        lds<4 * G>(t + L.v_codes() + lane * 4 * G, w0);
        lds<4 * G>(t + L.v_codes() + L.block() + lane * 4 * G, w1);
        lds<4 * G>(t + L.v_scales() + cc * 4 * G, vs0);
        lds<4 * G>(t + L.v_scales() + (cc + 4) * 4 * G, vs1);
        lds<2 * G>(t + L.v_zeros() + cc * 2 * G, vz0);
        lds<2 * G>(t + L.v_zeros() + (cc + 4) * 2 * G, vz1);
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          const uint32_t pick = grp & 1 ? 0x4342u : 0x4140u;  // 1024 + zero point of both tokens
          const uint32_t z0 = __byte_perm(vz0[grp >> 1], 0x64646464u, pick), z1 = __byte_perm(vz1[grp >> 1], 0x64646464u, pick);
          uint32_t v0[4], v1[4];
          v0[0] = code_pair<0>(w0[grp], 0x64006400u); v0[1] = code_pair<1>(w0[grp], 0x64006400u);
          v0[2] = code_pair<2>(w0[grp], 0x64006400u); v0[3] = code_pair<3>(w0[grp], 0x64006400u);
          v1[0] = code_pair<0>(w1[grp], 0x64006400u); v1[1] = code_pair<1>(w1[grp], 0x64006400u);
          v1[2] = code_pair<2>(w1[grp], 0x64006400u); v1[3] = code_pair<3>(w1[grp], 0x64006400u);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v0[j] = h2_mul(h2_sub(v0[j], z0), vs0[grp]);
            v1[j] = h2_mul(h2_sub(v1[j], z1), vs1[grp]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<false>(o[grp][0][nt], v0[0], v0[1], v1[0], v1[1], pb[tile][nt][0], pb[tile][nt][1]);
            mma16816<false>(o[grp][1][nt], v0[2], v0[3], v1[2], v1[3], pb[tile][nt][0], pb[tile][nt][1]);
          }
        }
      }
      __syncwarp();
      phase ^= 1u << stage;
      if (u + kStages * kWarps < u_end && !s_stop) issue(u + kStages * kWarps, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // ---- the warps' results become one
    __syncthreads();  // every copy has been waited for: the ring is free
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int k = 4; k <= 16; k <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], k);
        const int row = nt * 8 + 2 * cc + j;
        float* slab = merge + warp * C::kSlab + row * (D + 4);
#pragma unroll
        for (int grp = 0; grp < G; ++grp)
          *reinterpret_cast<float4*>(slab + grp * 32 + 4 * g) =
              make_float4(o[grp][0][nt][j], o[grp][0][nt][2 + j], o[grp][1][nt][j], o[grp][1][nt][2 + j]);
        if (g == 0) {
          slab[D] = m[nt][j];
          slab[D + 1] = l[nt][j];
        }
      }
    __syncthreads();

    const bool whole = seg_begin >= begin && seg_end <= end;
    const int cta0 = int(seg_begin / share), cta1 = int((seg_end - 1) / share);
    float* mine = p.partials + int64_t(2 * blockIdx.x + (seg_begin < begin ? 0 : 1)) * C::kPartial;
    auto put = [&](int row, int d, float v) {
      const int tok = (row0 + row) / a.group, h = head * a.group + (row0 + row) - tok * a.group;
      store_from_float(a.out, (s.first + tok) * a.o_ts + h * a.o_hs + d, a.dtype, v);
    };
    for (int i = tid; i < rows * D; i += kThreads) {
      const int row = i / D, d = i - row * D;
      float top = kNone, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge[w * C::kSlab + row * (D + 4) + D]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* slab = merge + w * C::kSlab + row * (D + 4);
        const float f = exp2f(slab[D] - top);
        sum = fmaf(f, slab[D + 1], sum);
        acc = fmaf(f, slab[d], acc);
      }
      if (whole) {
        put(row, d, sum == 0.f ? 0.f : acc / sum);
      } else {
        mine[row * D + d] = acc;
        if (d == 0) {
          mine[ROWS * D + row] = top;
          mine[ROWS * D + ROWS + row] = sum;
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int n = atomicAdd(p.counters + cta0, 1);
        s_last = n == cta1 - cta0;
        if (s_last) p.counters[cta0] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int i = tid; i < rows * D; i += kThreads) {
          const int row = i / D, d = i - row * D;
          float top = kNone, sum = 0.f, acc = 0.f;
          for (int k = cta0; k <= cta1; ++k) {
            const float* part = p.partials + int64_t(2 * k + (k == cta0 ? 1 : 0)) * C::kPartial;
            const float mk = __ldcg(part + ROWS * D + row), lk = __ldcg(part + ROWS * D + ROWS + row);
            const float ok = __ldcg(part + row * D + d), t = fmaxf(top, mk);
            const float f0 = exp2f(top - t), f1 = exp2f(mk - t);
            sum = sum * f0 + lk * f1;
            acc = acc * f0 + ok * f1;
            top = t;
          }
          put(row, d, sum == 0.f ? 0.f : acc / sum);
        }
      }
    }
    sm100::fence_proxy_async_smem();
    __syncthreads();  // before the ring, the fragments and the row table are written again
    at = seg_begin + (u_end - s.unit0);
  }
}

template <bool BF16, int G, int NT, bool MOD>
int launch_one(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  using C = Cfg<G, NT>;
  static PerContextOnce once;
  static int ctas_per_sm[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  auto kern = paged_attn_kernel<BF16, G, NT, MOD>;
  e = once.run(dev, [&] {
    cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (r == cudaSuccess) r = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas_per_sm[dev], kern, kThreads, C::kSmem);
    return r;
  });
  if (e != cudaSuccess) return cuda_status(e);
  AttnParams p;
  p.a = a;
  p.min_share = kWarps;
  p.max_rows = max_rows;
  const int64_t tiles = (std::min<int64_t>(int64_t(a.c.max_q) * a.group, max_rows) + C::ROWS - 1) / C::ROWS;
  const int64_t most = int64_t(a.c.batch) * a.c.kv_heads * tiles * ((a.c.limit + kUnit - 1) / kUnit + 1);
  const int64_t room = std::min<int64_t>(int64_t(device_sms(dev)) * std::max(1, ctas_per_sm[dev]), kMaxCtas);
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(room, (most + p.min_share - 1) / p.min_share));
  p.counters = static_cast<int*>(a.workspace);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kPagedCounterBytes);
  if (a.workspace_bytes < kPagedCounterBytes + size_t(grid) * 2 * C::kPartial * sizeof(float)) return SPECTRA_ERR_WORKSPACE;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

template <bool BF16, int G>
int launch_rows(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  const bool mod = a.softcap > 0.f || a.slopes;
  // up to 8 rows per key/value head: one column tile (fewer registers, more CTAs per SM); heads of 256 have
  // no registers for two
  if (G == 8 || int64_t(a.c.max_q) * a.group <= 8)
    return mod ? launch_one<BF16, G, 1, true>(a, max_rows, st) : launch_one<BF16, G, 1, false>(a, max_rows, st);
  constexpr int NT = G == 8 ? 1 : 2;
  return mod ? launch_one<BF16, G, NT, true>(a, max_rows, st) : launch_one<BF16, G, NT, false>(a, max_rows, st);
}

template <bool BF16>
int launch_dim(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 32: return launch_rows<BF16, 1>(a, max_rows, st);
    case 64: return launch_rows<BF16, 2>(a, max_rows, st);
    case 96: return launch_rows<BF16, 3>(a, max_rows, st);
    case 128: return launch_rows<BF16, 4>(a, max_rows, st);
    case 256: return launch_rows<BF16, 8>(a, max_rows, st);
  }
  return SPECTRA_ERR_UNSUPPORTED;
}

}  // namespace

size_t paged_attn_workspace_bytes(int head_dim) {
  return kPagedCounterBytes + size_t(kMaxCtas) * 2 * 16 * (head_dim + 2) * sizeof(float);
}

int launch_paged_attn(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  return a.dtype == SPECTRA_DT_BF16 ? launch_dim<true>(a, max_rows, st) : launch_dim<false>(a, max_rows, st);
}

int paged_attn_timeouts(long long* out, bool reset) { return read_timeout_counter(g_paged_attn_timeouts, out, reset); }

}  // namespace spectra
