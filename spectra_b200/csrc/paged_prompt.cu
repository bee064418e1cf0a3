// Attention over the paged INT4 KV cache for sm_100a: many new tokens of a
// sequence (prompts, chunks of prompts), on the tcgen05 tensor cores.
//
// The definition is paged_attn.cu's.  With hundreds of rows per key/value head
// the work is products, so a CTA takes 256 rows (tokens x the query heads that
// share the head; two M = 128 tiles, one for heads of 256) of one sequence and
// walks the keys 64 at a time, the last ones first: the step with the causal
// edge is then the one that has to look for a maximum anyway, and a bias on
// distance only falls afterwards.
//   warps 8-11  bring the raw tiles in by bulk copies and write them to shared
//               memory as fp16 operands: K [token][feature] and V^T
//               [feature][token], K-major, 128-byte swizzle; two warps a step,
//               in turn.  (q - z) s is an exact difference and one rounding (11 bits),
//               or two exact operands (Cfg).
//   warps 12, 13  S_t = Q_t K^T (Q in shared memory) and O_t += P_t V (P in
//               TMEM), t = 0, 1.  Each tile has two S buffers, so the scores of
//               the next step are there when a softmax ends.
//   warps 0-7   one row per thread: scores from TMEM, P back to TMEM over
//               them as fp16, running maximum and sum in registers.  The
//               maximum is raised only when the weights it gives grow large;
//               then (rarely after the first step) O is rescaled in TMEM.
// The features of Q and K, and the tokens of P and V, are contracted in the
// order in which the codes unpack.  bf16 queries are scaled by a power of two
// per row to fit fp16, so only differences below 2^-28 of a row's largest
// entry are lost.
// TMEM (512 columns): S_0 (two buffers) | S_1 (two) | O_0 | O_1.
//
// With fewer CTAs than SMs the keys are split over `splits` CTAs per tile,
// whose partial results a second small kernel puts together.
//
// Rounded to fp16's 11 bits: queries (fp16: not at all, bf16: only as said),
// keys and values (except where Cfg has two operands), because fp16 operands run
// at the full tensor rate and the codes carry 4 bits; weights, kept times 2^kShift
// so that small ones are not subnormal (below 2^-28 of the largest they are lost
// from O, not from their sum).  Scores, maxima, sums and outputs stay in fp32.
//
// Measured: 4096 tokens over 16384, 32 query heads on 8, heads of 128, 1101 us
// (874 TFLOP/s over the visible pairs); a prompt of 1024 tokens 31 us; 6 ragged
// prompts up to 2501 with a cap, 64 query heads on 8, heads of 64, fp16, 448 us.
// Bound by the softmax warps (one exponential a score on the special-function
// unit, and their issue slots) with the tensor pipe close behind; short prompts
// and small heads also by what a step waits for and by instruction fetches.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "gemv_mma.cuh"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

__device__ int g_paged_prompt_timeouts = 0;

namespace {

using namespace sm100;

constexpr int kRows = 256;   // rows of a CTA, at most
constexpr int kKeys = 64;    // keys of a step
constexpr uint32_t kUpper = 0xFFF0FFF0u;  // of two fp16 numbers: sign, exponent, 7 bits
constexpr int kThreads = 512;  // warps 14 and 15 only give their registers away

struct PromptParams {
  PagedAttnArgs a;
  int row_tiles;   // per sequence and head, at most
  int splits;
  int rows;        // of a CTA
  int min_rows;    // a sequence with at most this many rows per head is the other kernel's
  float* partials; // [item][split][rows][D + 2]
};

// Keys and values in one operand are rounded to 11 bits, which alone puts results 7e-4 off (keys of
// loud features) where an fp16 result's own rounding is 2.0e-4.  fp16 queries of heads up to 64 take
// them as two, (q - z) s_hi + (q - z) s_lo with the scale's upper 7 bits and the rest: exact in fp16.
// That is twice the products, for which the tensor pipe has room there (6 capped prompts, heads of 64,
// 448 us against 408, plain ones 162 against 145) and no longer with heads of 128 (258 us against 180;
// a chunk of 4096 over 16384 1800 against 1033) or 256; a bf16 result has 1.6e-3 of its own.
template <int G, bool BF16>
struct Cfg {
  static constexpr int D = 32 * G;
  static constexpr int kAtoms = (D + 63) / 64;                 // 128-byte column blocks of Q and K
  static constexpr int kTile = TileLayout{G}.bytes();
  static constexpr int kQAtom = 128 * 128;                     // 128 rows
  static constexpr int kKAtom = kKeys * 128;                   // 64 rows
  // Heads of 256: O takes 256 columns of TMEM and a step's operands 64 KB, so one tile, two stages of
  // keys and one of values.
  static constexpr int kTiles = G == 8 ? 1 : 2;
  static constexpr int kParts = !BF16 && G <= 2 ? 2 : 1;       // operands
  static constexpr int kKStages = (G == 8 ? 2 : 4) / kParts, kVStages = G == 8 ? 1 : 4 / kParts;
  static constexpr int kQ = kTiles * kAtoms * kQAtom;
  static constexpr int kKPart = kAtoms * kKAtom, kVPart = D * 128;
  static constexpr int kK = kParts * kKPart, kV = kParts * kVPart;  // one stage
  static constexpr int kRaw = 4 * 2 * kTile;
  static constexpr int kSmem = 1024 + kQ + kKStages * kK + kVStages * kV + kRaw;
};

// The rows of one item: row R of a (sequence, head) is token R / group, query head R % group.
struct Item {
  int b, head, row0, rows;
  int64_t first;
  int pos0, len;
  int step0, steps;  // of this CTA's share of the keys, kKeys each
};

__device__ __forceinline__ bool item_of(const PromptParams& p, int index, int split, Item& it) {
  const PagedView& c = p.a.c;
  const int per = c.batch * c.kv_heads;
  const int tile = p.row_tiles - 1 - index / per;  // the longest first
  const int bh = index % per;
  it.head = bh % c.kv_heads;
  it.b = bh / c.kv_heads;
  int count, extra;
  new_rows(c, it.b, it.first, count, extra);
  const int all = count * p.a.group;
  it.row0 = tile * p.rows;
  if (all <= p.min_rows || it.row0 >= all) return false;
  it.rows = min(p.rows, all - it.row0);
  const int len = c.seq_lens[it.b];
  it.pos0 = len - count - extra;
  it.len = len < 0 ? 0 : (len < c.limit ? len : c.limit);
  const int p0 = it.pos0 + it.row0 / p.a.group, p1 = it.pos0 + (it.row0 + it.rows - 1) / p.a.group;
  const int hi = p1 < 0 ? 0 : (p.a.causal ? min(it.len, p1 + 1) : it.len);
  const int lo = first_key(p0, p.a.window);
  const int s0 = lo / kKeys, s1 = (hi + kKeys - 1) / kKeys;
  const int n = hi > lo ? s1 - s0 : 0;
  it.step0 = s0 + int((int64_t(n) * split) / p.splits);
  it.steps = s0 + int((int64_t(n) * (split + 1)) / p.splits) - it.step0;
  return true;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld_x32_nowait(taddr, r);
  tmem_ld_wait32(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// MOD: 0 plain scores, 1 with a cap of up to kLowCap, 2 with a bias (and a cap where softcap > 0) or a
// higher cap (whose code in MOD 1 took 490 us where 450 are taken without it)
template <bool BF16, int G, int MOD>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(PromptParams p) {
  using C = Cfg<G, BF16>;
  constexpr int D = C::D;
  constexpr TileLayout L{G};
  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sk = sq + C::kQ;
  uint8_t* sv = sk + C::kKStages * C::kK;
  uint8_t* raw = sv + C::kVStages * C::kV;
  // (the values' stages are freed on two barriers at least: the warps of the odd and of the even steps
  // each see every phase of the one they wait on)
  constexpr int SK = C::kKStages, SV = C::kVStages, SE = SV == 1 ? 2 : SV;
  __shared__ uint64_t q_full, k_full[SK], v_full[SV], k_empty[SK], v_empty[SE];
  __shared__ uint64_t s_full[2][2], p_full[2][2], o_full[2], o_done[2], raw_full[4], drain[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_held[8][2];  // [step % 8][half]: which of the half's two tiles a page holds
  __shared__ volatile int s_abort, s_never;

  // what a whole warp agrees on comes out of a shuffle, which tells the compiler so: the
  // products' operands then stay in uniform registers
  auto same = [](auto v) { return __shfl_sync(0xffffffffu, v, 0); };
  const int tid = threadIdx.x, warp = same(tid >> 5), lane = tid & 31;
  const int split = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  Item it;
  if (!item_of(p, blockIdx.x, split, it)) return;
  const int tiles = same(it.rows > 128 ? 2 : 1);
  if (tid == 0) {
    mbar_init(&q_full, 8);
    for (int i = 0; i < SK; ++i) {
      mbar_init(k_full + i, 2);
      mbar_init(k_empty + i, tiles);
    }
    for (int i = 0; i < SV; ++i) mbar_init(v_full + i, 2);
    for (int i = 0; i < SE; ++i) mbar_init(v_empty + i, tiles);
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&s_full[i][j], 1);
        mbar_init(&p_full[i][j], 4);
      }
      mbar_init(o_full + i, 1);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(raw_full + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(drain + i, 1);
    s_abort = s_never = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = same(s_tmem);
  const int n = same(it.steps);

  // A whole warp waits, and the vote makes its lanes agree: one may see a phase complete, or the
  // abort, a poll later than the next, and lanes that part here would miss each other at the votes
  // and the warp-wide TMEM accesses that follow.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, mbar_wait_inline(bar, parity, &s_abort))) return true;
    if (!s_abort) {
      s_abort = 1;
      if (lane == 0) atomicAdd(&g_paged_prompt_timeouts, 1);
    }
    return false;
  };

  // Registers by role: 2 x 128 x 152 + 128 x 128 (unchanged) + 128 x 80 = the launch's 512 x 128.
  if (warp < 8) {
    // ------------------------------------------------------------ rows
    reg_inc<152>();
    const int t = warp >> 2, row = tid & 127, r = t * 128 + row;
    const bool real = r < it.rows;
    const int R = it.row0 + r, tok = real ? R / a.group : 0;
    const int h = it.head * a.group + (real ? R - tok * a.group : 0);
    const int pos = it.pos0 + tok;
    float c_row = a.scale;
    // rows of 16-byte chunks, swizzled: the query operand, and later the result; kLanes lanes bring a row
    constexpr int kChunks = D / 8, kLanes = G == 3 ? 16 : kChunks, kPer = 32 / kLanes;
    const int w0 = (warp & 3) * 32;
    uint8_t* q_tile = sq + t * C::kAtoms * C::kQAtom;
    auto chunk_at = [&](int r, int ch) { return q_tile + (ch / 8) * C::kQAtom + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
    const int ch = lane & (kLanes - 1);
    if (t < tiles) {
      // The warp's 32 queries to where their operand will be, whole rows at a time (a lane brings 16
      // bytes of one; row by row per thread, each load would touch 32 lines) ...
      const uint16_t* mine = reinterpret_cast<const uint16_t*>(a.q) + (it.first + tok) * a.q_ts + h * a.q_hs;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += kPer) {
        const int r = r0 + lane / kLanes;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(mine), r)) + 8 * ch;
        const bool have = t * 128 + w0 + r < it.rows;
        if (ch < kChunks) {
          uint8_t* dst = chunk_at(w0 + r, ch);
          if (a.vec) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(have ? src : mine), "r"(have ? 16 : 0)
                         : "memory");
          } else {
            uint32_t u[4] = {};
            if (have) {
#pragma unroll
              for (int j = 0; j < 4; ++j) u[j] = uint32_t(src[2 * j]) | (uint32_t(src[2 * j + 1]) << 16);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      // ... then each thread its row, in place: scaled to fp16, features in the order (0,4)(1,5)(2,6)(3,7)
      float f = 1.f;
      if constexpr (BF16) {
        uint32_t top2 = 0;
#pragma unroll 4
        for (int i = 0; i < kChunks; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(chunk_at(row, i));
          top2 = max_abs2<true>(max_abs2<true>(max_abs2<true>(max_abs2<true>(top2, v.x), v.y), v.z), v.w);
        }
        const uint32_t top = max(top2 >> 16, top2 & 0xFFFFu) >> 7;  // largest exponent
        // largest entry to [2^4, 2^5) (an infinity or NaN: as it is); both factors stay normal numbers
        const int e = min(top == 255u ? 0 : 131 - int(top), 100);
        f = __uint_as_float(uint32_t(127 + e) << 23);
        c_row *= __uint_as_float(uint32_t(127 - e) << 23);
      }
#pragma unroll 4
      for (int i = 0; i < kChunks; ++i) {
        uint4* at = reinterpret_cast<uint4*>(chunk_at(row, i));
        uint32_t w[4] = {at->x, at->y, at->z, at->w};
        if constexpr (BF16) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = h2_pack(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xFFFF0000u) * f);
        }
        *at = make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x5410),
                         __byte_perm(w[1], w[3], 0x7632));
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full);

    if (t < tiles) {
      int hi = 0x7FFFFFFF, lo = 0;  // keys this row sees
      if (real) {
        hi = pos < 0 ? 0 : (a.causal ? min(it.len, pos + 1) : it.len);
        lo = first_key(pos, a.window);
      }
      const float slope = MOD == 2 && a.slopes ? a.slopes[h] * kLog2e : 0.f;
      const float inv = MOD != 0 && a.softcap > 0.f ? cap_factor(c_row, a.softcap) : 0.f;
      const float k_exp = c_row * kLog2e;
      const uint32_t quarter = uint32_t((warp & 3) * 32) << 16;
      const uint32_t to = tmem + quarter + 256 + t * 128;
      float m = kNone, l = 0.f;
      bool ok = true, loud = false;  // loud: a maximum past kLoud

      for (int i = 0; i < n; ++i) {
        const uint32_t ts = tmem + quarter + t * 128 + (i & 1) * 64;
        ok = wait(&s_full[t][i & 1], (i >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const int n0 = (it.step0 + n - 1 - i) * kKeys;
        const int held = s_held[i & 7][0] | s_held[i & 7][1] << 2;  // one bit per 16 keys
        const bool masked = __any_sync(0xffffffffu, n0 < lo || n0 + kKeys > hi) || held != 0xF;

        // Most steps: no mask, no new maximum.  The weights are computed with the old maximum and
        // stored if their sum is small enough to say that no score passed it by much (then each
        // weight fits fp16 too) and no score is out of the range of the cap's tanh.  (A second copy with
        // four of its six terms, for steps of low scores, cost more in instruction fetches than it saved:
        // heads of 64, 6 ragged prompts, 477 us against 426; heads of 128, 234 against 238.)
        auto fast = [&](auto cap) -> bool {
          constexpr bool CAP = decltype(cap)::value;
          constexpr float kMost = 61440.f;  // fits fp16, with 6 % for the sum's own error
          uint32_t buf[2][32], pk[32];
          uint64_t sums[2] = {0, 0}, fit[6];
          float far = 0.f;
          const uint64_t m2 = f2(kShift - m, kShift - m);
          const float c1 = CAP ? inv : k_exp;
          const uint64_t first = f2(c1, c1);
          if constexpr (CAP) {
#pragma unroll
            for (int d = 0; d < 6; ++d) {
              const float x = a.softcap * kLog2e * kTanhFit6[d];
              fit[d] = f2(x, x);
            }
          }
          tmem_ld_x32_nowait(ts, buf[0]);
          tmem_ld_wait32(buf[0]);
          tmem_ld_x32_nowait(ts + 32, buf[1]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q == 1) tmem_ld_wait32(buf[1]);
            const uint32_t(&v)[32] = buf[q];
            [[maybe_unused]] const float bias = MOD == 2 ? slope * float(n0 + 32 * q - pos) + (kShift - m) : 0.f;
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const uint64_t raw2 = f2(__uint_as_float(v[k]), __uint_as_float(v[k + 1]));
              uint64_t y = m2;
              if constexpr (MOD == 2) y = f2_fma(f2(slope, slope), f2(float(k), float(k + 1)), f2(bias, bias));
              if constexpr (!CAP) {
                y = f2_fma(raw2, first, y);
              } else {
                const uint64_t x = f2_mul(raw2, first), u = f2_mul(x, x);
                float u0, u1;
                f2_split(u, u0, u1);
                far = max3(far, u0, u1);
                uint64_t r = fit[5];
#pragma unroll
                for (int d = 4; d >= 0; --d) r = f2_fma(r, u, fit[d]);
                y = f2_fma(x, r, y);
              }
              float e0, e1;  // exponents: scores in powers of two, less the maximum
              f2_split(y, e0, e1);
              e0 = ex2(e0);
              e1 = ex2(e1);
              sums[(k >> 1) & 1] = f2_add(sums[(k >> 1) & 1], f2(e0, e1));
              // pairs in the order of the value operand's tokens
              pk[16 * q + 4 * ((k >> 1) & 3) + (k >> 3)] = h2_pack(e0, e1);
            }
          }
          float s0, s1;
          f2_split(f2_add(sums[0], sums[1]), s0, s1);
          s0 += s1;
          if (__any_sync(0xffffffffu, s0 > kMost || (CAP && far > kTanhRange6))) return false;
          l += s0;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t u[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) u[k] = pk[16 * q + k];
            tmem_st_x16(ts + 16 * q, u);
          }
          return true;
        };
        bool done = false;
        if (i > 0 && !masked && !loud) {
          if constexpr (MOD == 0)
            done = fast(std::false_type{});
          else if (MOD == 2 && !(a.softcap > 0.f))
            done = fast(std::false_type{});
          else
            done = fast(std::true_type{});
        }
        if (!done) {
          uint32_t buf[2][32];
          tmem_ld_x32_nowait(ts, buf[0]);
          tmem_ld_x32_nowait(ts + 32, buf[1]);
          tmem_ld_wait32(buf[0]);
          tmem_ld_wait32(buf[1]);
          if (MOD == 2 && a.softcap > kLowCap) {
            const float back = 1.f / inv;
#pragma unroll
            for (int k = 0; k < 64; ++k) {
              uint32_t& w = buf[k >> 5][k & 31];
              w = __float_as_uint(high_cap(__uint_as_float(w), inv, back));
            }
          }
          const bool low_cap = MOD == 1 || (a.softcap > 0.f && a.softcap <= kLowCap);
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < 64; ++k) {
            uint32_t& w = buf[k >> 5][k & 31];
            float x = __uint_as_float(w);
            if constexpr (MOD == 0) {
              x *= k_exp;
            } else {
              x = low_cap ? a.softcap * tanh_exp(x * inv) : x * c_row;
              x = fmaf(slope, float(n0 + k - pos), x * kLog2e);
            }
            if (masked) x = n0 + k >= hi || n0 + k < lo || !((held >> (k / 16)) & 1) ? -INFINITY : x;
            w = __float_as_uint(x);
            top = fmaxf(top, x);
          }
          // (after this no weight of this step passes 2^(3 + kShift): sums like it stay in fast's bound)
          if (__any_sync(0xffffffffu, top > m + 3.f)) {
            const float up = fmaxf(m, top), f = exp2f(m - up);
            m = up;
            loud = __any_sync(0xffffffffu, fabsf(m) > kLoud);
            l *= f;
            if (i > 0) {  // O, once the last step's product has been added
              ok = wait(o_full + t, (i - 1) & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int d = 0; d < D; d += 32) {
                float v[32];
                tmem_ld32(to + d, v);
                uint32_t u[16];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
                  for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(v[16 * hh + k] * f);
                  tmem_st_x16(to + d + 16 * hh, u);
                }
              }
            }
          }
          float sum[4] = {};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t u[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float e0 = ex2(__uint_as_float(buf[q][k]) + (kShift - m));
              const float e1 = ex2(__uint_as_float(buf[q][k + 1]) + (kShift - m));
              sum[k & 2] += e0;
              sum[(k & 2) + 1] += e1;
              u[4 * ((k >> 1) & 3) + (k >> 3)] = h2_pack(e0, e1);
            }
            tmem_st_x16(ts + 16 * q, u);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t][i & 1]);
      }

      // ---- result
      if (n > 0 && ok) ok = wait(o_done + t, 0);
      tc_fence_after();
      if (p.splits > 1) {
        float* part = p.partials + ((int64_t(blockIdx.x) * p.splits + split) * p.rows + r) * (D + 2);
#pragma unroll
        for (int d = 0; d < D; d += 32) {
          float v[32];
          if (n > 0) tmem_ld32(to + d, v);
          if (real) {
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              *reinterpret_cast<float2*>(part + d + k) = n > 0 ? make_float2(v[k], v[k + 1]) : make_float2(0.f, 0.f);
          }
        }
        if (real) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
      } else {
        // through shared memory (this tile's queries are no longer needed), so that whole rows are stored
        const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          float v[32];
          if (n > 0) tmem_ld32(to + d, v);
          uint32_t u[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float x = l == 0.f ? 0.f : v[2 * k] * f, y = l == 0.f ? 0.f : v[2 * k + 1] * f;
            if constexpr (BF16) {
              const __nv_bfloat162 b2 = __floats2bfloat162_rn(x, y);
              u[k] = *reinterpret_cast<const uint32_t*>(&b2);
            } else {
              u[k] = h2_pack(x, y);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(chunk_at(row, d / 8 + k)) = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
        }
        __syncwarp();
        const uint64_t mine = reinterpret_cast<uint64_t>(reinterpret_cast<uint16_t*>(a.out) + (it.first + tok) * a.o_ts + h * a.o_hs);
#pragma unroll 4
        for (int r0 = 0; r0 < 32; r0 += kPer) {
          const int rr = r0 + lane / kLanes;
          uint16_t* dst = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, mine, rr)) + 8 * ch;
          if (ch < kChunks && t * 128 + w0 + rr < it.rows) {
            const uint4 v = *reinterpret_cast<const uint4*>(chunk_at(w0 + rr, ch));
            if (a.vec) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int k = 0; k < 8; ++k) dst[k] = uint16_t(u[k >> 1] >> (16 * (k & 1)));
            }
          }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ operands
    // warps 8 and 9 take steps 0, 2, ..., warps 10 and 11 steps 1, 3, ...; each 32 of a step's keys
    const int dw = warp - 8, g = lane >> 2, cc = lane & 3, half = dw & 1;
    uint8_t* buf = raw + dw * 2 * C::kTile;
    const uint32_t magic = fp16_1024();
    int mine = 0;            // lanes 0, 1: page of the tile to load next
    auto look = [&](int i) {
      const int at = (it.step0 + n - 1 - i) * kKeys + 32 * half + 16 * lane;
      mine = lane < 2 && i < n && at < it.len ? c.tables[it.b * c.table_stride + (at >> c.page_log2)] : -1;
    };
    unsigned held_next = 0;  // lanes 0, 1: of the tiles in flight
    auto issue = [&](int i) {
      if (lane < 2) {
        const bool hold = unsigned(mine) < unsigned(c.num_pages);
        held_next = __ballot_sync(0x3u, hold);
        if (lane == 0) mbar_arrive_expect_tx(raw_full + dw, __popc(held_next) * C::kTile);
        __syncwarp(0x3u);
        if (hold) {
          const int at = (it.step0 + n - 1 - i) * kKeys + 32 * half + 16 * lane;
          const int per = 1 << (c.page_log2 - 4);
          bulk_g2s(buf + lane * C::kTile, c.pool + mine * c.page_stride + (int64_t(it.head) * per + ((at >> 4) & (per - 1))) * C::kTile,
                   C::kTile, raw_full + dw);
        }
      }
    };
    const int first = dw >> 1;
    if (first < n) {
      look(first);
      issue(first);
      look(first + 2);
    }
    bool ok = true, flying = false;  // a copy that nothing has waited for, and its phase
    uint32_t phase = 0;
    // Heads of 256 have no registers for a whole step: their values are read after the keys are done,
    // and the next copy waits for that.
    constexpr bool kLate = G == 8;
    for (int i = first; i < n; i += 2) {
      const int sk_at = i % SK, sv_at = i % SV;
      const unsigned held = __shfl_sync(0xffffffffu, held_next, 0);
      flying = false;
      if (!__all_sync(0xffffffffu, mbar_wait_inline(raw_full + dw, phase, &s_never))) {  // (its own copy: waited for whatever the others saw)
        if (lane == 0) atomicAdd(&g_paged_prompt_timeouts, 1);
        s_abort = 1;
        break;
      }
      phase ^= 1;
      uint32_t kw[2][2][G], vw[2][2][G], ks[2][2][(2 * G + 3) / 4], kz[2][2][(G + 3) / 4], vs[2][2][G], vz[2][2][(2 * G + 3) / 4];
      auto values = [&]() {  // and the next step's copy
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint8_t* tp = buf + x * C::kTile;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            lds<4 * G>(tp + L.v_codes() + y * L.block() + lane * 4 * G, vw[x][y]);
            lds<4 * G>(tp + L.v_scales() + (cc + 4 * y) * 4 * G, vs[x][y]);
            lds<2 * G>(tp + L.v_zeros() + (cc + 4 * y) * 2 * G, vz[x][y]);
          }
          if (!((held >> x) & 1u)) {  // no page: keys are masked, values have to be finite
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int q = 0; q < G; ++q) vs[x][y][q] = 0;
          }
        }
        __syncwarp();
        flying = i + 2 < n;
        if (flying) {
          issue(i + 2);
          look(i + 4);
        }
      };
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* tp = buf + x * C::kTile;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          lds<4 * G>(tp + L.k_codes() + y * L.block() + lane * 4 * G, kw[x][y]);
          lds<2 * G>(tp + L.k_scales() + (g + 8 * y) * 2 * G, ks[x][y]);
          lds<G>(tp + L.k_zeros() + (g + 8 * y) * G, kz[x][y]);
        }
      }
      if constexpr (!kLate) values();

      // ---- keys: [token][feature]
      if (i >= SK) ok = wait(k_empty + sk_at, (i / SK - 1) & 1);
      if (!ok) break;
      if (lane == 0) s_held[i & 7][half] = int(held);
      uint8_t* kd = sk + sk_at * C::kK;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int q = 0; q < G; ++q) {
            const uint32_t s2 = __byte_perm(ks[x][y][q >> 1], 0, q & 1 ? 0x3232 : 0x1010);
            const uint32_t b = q & 3, z2 = __byte_perm(kz[x][y][q >> 2], 0x64646464u, b | 0x40u | (b << 8) | 0x4000u);
            const uint32_t c2 = h2_sub(0x63806380u, z2);  // 960 - (1024 + z)
            const uint32_t w = kw[x][y][q];
            const uint32_t d0 = h2_sub(code_low(w, magic), z2), d1 = h2_fma(code_high(w, magic), 0x2C002C00u, c2),
                           d2 = h2_sub(code_low(w >> 8, magic), z2), d3 = h2_fma(code_high(w >> 8, magic), 0x2C002C00u, c2);
            const int row = 32 * half + 16 * x + 8 * y + g;
            uint8_t* at = kd + (q >> 1) * C::kKAtom + row * 128 + ((((q & 1) * 4 + cc) ^ g) << 4);
            const uint32_t hi = C::kParts == 2 ? s2 & kUpper : s2;
            *reinterpret_cast<uint4*>(at) = make_uint4(h2_mul(d0, hi), h2_mul(d1, hi), h2_mul(d2, hi), h2_mul(d3, hi));
            if constexpr (C::kParts == 2) {
              const uint32_t lo = h2_sub(s2, hi);
              *reinterpret_cast<uint4*>(at + C::kKPart) = make_uint4(h2_mul(d0, lo), h2_mul(d1, lo), h2_mul(d2, lo), h2_mul(d3, lo));
            }
          }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_full + sk_at);
      if constexpr (kLate) values();

      // ---- values: [feature][token], tokens {2c, 2c+1, 2c+8, 2c+9, 2c+16, ...} of the 32 as chunk c
      if (i >= SV) ok = wait(v_empty + (i - SV) % SE, ((i - SV) / SE) & 1);
      if (!ok) break;
      uint8_t* vd = sv + sv_at * C::kV;
#pragma unroll
      for (int q = 0; q < G; ++q) {
        uint32_t o[4][4];
        [[maybe_unused]] uint32_t rest[4][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t z2 = byte_pair(vz[x][y][q >> 1], q & 1), c2 = h2_sub(0x63806380u, z2);
            const uint32_t w = vw[x][y][q], s2 = vs[x][y][q];
            const uint32_t d[4] = {h2_sub(code_low(w, magic), z2), h2_fma(code_high(w, magic), 0x2C002C00u, c2),
                                   h2_sub(code_low(w >> 8, magic), z2), h2_fma(code_high(w >> 8, magic), 0x2C002C00u, c2)};
            const uint32_t hi = C::kParts == 2 ? s2 & kUpper : s2;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[j][2 * x + y] = h2_mul(d[j], hi);
              if constexpr (C::kParts == 2) rest[j][2 * x + y] = h2_mul(d[j], h2_sub(s2, hi));
            }
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 32 * q + 4 * g + j;
          uint8_t* at = vd + row * 128 + (((half * 4 + cc) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = make_uint4(o[j][0], o[j][1], o[j][2], o[j][3]);
          if constexpr (C::kParts == 2)
            *reinterpret_cast<uint4*>(at + C::kVPart) = make_uint4(rest[j][0], rest[j][1], rest[j][2], rest[j][3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_full + sv_at);
    }
    if (flying && !ok) mbar_wait_inline(raw_full + dw, phase, &s_never);
  } else {
    reg_dec<80>();
  }
  if (warp >= 12 && warp < 12 + tiles && n > 0) {
    // ------------------------------------------------------------ products, a warp for each tile
    constexpr uint32_t id_s = idesc_f16(false, 128, kKeys), id_o = idesc_f16(false, 128, D);
    const uint32_t one = elect_one();
    const int t = warp - 12;
    const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * 128;
    const uint64_t dq = smem_desc_k_sw128(smem_u32(sq) + t * C::kAtoms * C::kQAtom), dk = smem_desc_k_sw128(smem_u32(sk)),
                   dv = smem_desc_k_sw128(smem_u32(sv));
    // (descriptors count in 16 bytes)
    auto scores = [&](int i) {
#pragma unroll
      for (int part = 0; part < C::kParts; ++part)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss_one(ts + (i & 1) * 64, dq + (((k / 4) * C::kQAtom + (k % 4) * 32) >> 4),
                     dk + (((i % SK) * C::kK + part * C::kKPart + (k / 4) * C::kKAtom + (k % 4) * 32) >> 4), id_s,
                     part > 0 || k > 0, one);
      mma_commit_one(&s_full[t][i & 1], one);
      mma_commit_one(k_empty + i % SK, one);
    };
    bool ok = wait(&q_full, 0);
    for (int i = 0; i < 2 && i < n && ok; ++i) {
      ok = wait(k_full + i, 0);  // (two stages at least)
      tc_fence_after();
      if (ok) scores(i);
    }
    for (int i = 0; i < n && ok; ++i) {
      ok = wait(v_full + i % SV, (i / SV) & 1) && wait(&p_full[t][i & 1], (i >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int part = 0; part < C::kParts; ++part)
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_ts_one(to, ts + (i & 1) * 64 + k * 8, dv + (((i % SV) * C::kV + part * C::kVPart + k * 32) >> 4), id_o,
                     i > 0 || part > 0 || k > 0, one);
      mma_commit_one(o_full + t, one);
      mma_commit_one(v_empty + i % SE, one);
      if (i + 1 == n) mma_commit_one(o_done + t, one);
      if (i + 2 < n) {
        // its weights have been read: scores may take their place
        ok = wait(k_full + (i + 2) % SK, ((i + 2) / SK) & 1) && wait(o_full + t, i & 1);
        if (!ok) break;
        tc_fence_after();
        scores(i + 2);
      }
    }
    if (!ok) {  // products that are still running read shared memory and TMEM
      mma_commit_one(drain + t, one);
      mbar_wait_inline(drain + t, 0, &s_never);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp per row: the partial results of its splits.
template <bool BF16, int G>
__global__ void __launch_bounds__(256) paged_prompt_join_kernel(PromptParams p) {
  constexpr int D = 32 * G;
  pdl_wait();
  pdl_trigger();
  const PagedAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  Item it;
  if (!item_of(p, blockIdx.x, 0, it)) return;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= it.rows) return;
  const float* part = p.partials + (int64_t(blockIdx.x) * p.splits * p.rows + r) * (D + 2);
  const int64_t step = int64_t(p.rows) * (D + 2);
  float top = kNone, sum = 0.f, acc[G];
#pragma unroll
  for (int q = 0; q < G; ++q) acc[q] = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 32) {  // 32 splits' weights at once, then eight splits' loads in flight
    const bool in = s0 + lane < p.splits;
    const float2 ml = in ? *reinterpret_cast<const float2*>(part + (s0 + lane) * step + D) : make_float2(kNone, 0.f);
    float up = fmaxf(top, ml.x);
#pragma unroll
    for (int k = 16; k; k >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, k));
    const float fade = exp2f(top - up), f = in ? exp2f(ml.x - up) : 0.f;
    float more = f * ml.y;
#pragma unroll
    for (int k = 16; k; k >>= 1) more += __shfl_xor_sync(0xffffffffu, more, k);
    top = up;
    sum = fmaf(sum, fade, more);
#pragma unroll
    for (int q = 0; q < G; ++q) acc[q] *= fade;
    const int n = min(32, p.splits - s0);
    for (int s = 0; s < n; s += 8) {
      float v[8][G];
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int q = 0; q < G; ++q) v[x][q] = part[(s0 + min(s + x, n - 1)) * step + 32 * q + lane];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float w = __shfl_sync(0xffffffffu, f, (s + x) & 31);
#pragma unroll
        for (int q = 0; q < G; ++q) acc[q] = s + x < n ? fmaf(w, v[x][q], acc[q]) : acc[q];
      }
    }
  }
  const int R = it.row0 + r, tok = R / a.group, h = it.head * a.group + R - tok * a.group;
#pragma unroll
  for (int q = 0; q < G; ++q)
    store_from_float(a.out, (it.first + tok) * a.o_ts + h * a.o_hs + 32 * q + lane, a.dtype, sum == 0.f ? 0.f : acc[q] / sum);
}

template <class K>
int launch_dep(K kernel, dim3 grid, int threads, int smem, const PromptParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p));
}

template <bool BF16, int G, int MOD>
int launch_one(const PagedAttnArgs& a, int min_rows, cudaStream_t st) {
  using C = Cfg<G, BF16>;
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  auto kern = paged_prompt_kernel<BF16, G, MOD>;
  e = once.run(dev, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem); });
  if (e != cudaSuccess) return cuda_status(e);
  PromptParams p;
  p.a = a;
  p.min_rows = min_rows;
  p.rows = 128 * C::kTiles;
  p.row_tiles = int((int64_t(a.c.max_q) * a.group + p.rows - 1) / p.rows);
  const int64_t items = int64_t(p.row_tiles) * a.c.batch * a.c.kv_heads;
  if (items > INT32_MAX) return SPECTRA_ERR_SHAPE;
  // four steps of keys a split at least
  const int64_t most = std::max<int64_t>(1, a.c.limit / (4 * kKeys));
  p.splits = int(std::max<int64_t>(1, std::min<int64_t>(most, device_sms(dev) / items)));
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kPagedCounterBytes);
  if (p.splits > 1 &&
      a.workspace_bytes < kPagedCounterBytes + size_t(items) * p.splits * p.rows * (C::D + 2) * sizeof(float))
    return SPECTRA_ERR_WORKSPACE;
  const int status = launch_dep(kern, dim3(unsigned(items), unsigned(p.splits)), kThreads, C::kSmem, p, st);
  if (status != SPECTRA_OK || p.splits == 1) return status;
  return launch_dep(paged_prompt_join_kernel<BF16, G>, dim3(unsigned(items), unsigned(p.rows / 8)), 256, 0, p, st);
}

template <bool BF16, int G>
int launch_mod(const PagedAttnArgs& a, int min_rows, cudaStream_t st) {
  if (a.slopes || a.softcap > kLowCap) return launch_one<BF16, G, 2>(a, min_rows, st);
  return a.softcap > 0.f ? launch_one<BF16, G, 1>(a, min_rows, st) : launch_one<BF16, G, 0>(a, min_rows, st);
}

template <bool BF16>
int launch_dim(const PagedAttnArgs& a, int min_rows, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 32: return launch_mod<BF16, 1>(a, min_rows, st);
    case 64: return launch_mod<BF16, 2>(a, min_rows, st);
    case 96: return launch_mod<BF16, 3>(a, min_rows, st);
    case 128: return launch_mod<BF16, 4>(a, min_rows, st);
    case 256: return launch_mod<BF16, 8>(a, min_rows, st);
  }
  return SPECTRA_ERR_UNSUPPORTED;
}

}  // namespace

size_t paged_prompt_workspace_bytes(int head_dim) {
  // (splits only while items * splits <= SMs; 160 covers every sm_100a part)
  return kPagedCounterBytes + size_t(160) * kRows * (head_dim + 2) * sizeof(float);
}

int launch_paged_prompt(const PagedAttnArgs& a, int min_rows, cudaStream_t st) {
  return a.dtype == SPECTRA_DT_BF16 ? launch_dim<true>(a, min_rows, st) : launch_dim<false>(a, min_rows, st);
}

// Rows of one key/value head (new tokens times the query heads that share it): up to `few` a
// sequence is paged_attn.cu's, above it this file's.  A batch of equal sequences takes one
// launch; a ragged one with long sequences both, as either kind may be in it.  Measured with
// heads of 128, 8 of them, 32 queries' heads, us (paged_attn / paged_prompt):
//   keys   1 sequence, 64 rows   96 rows       16 sequences, 32 rows   64 rows
//   1024   13.3 / 17.1           19.4 / 18.2   27.7 / 25.1             44.3 / 25.8
//   8192   27.9 / 33.5           33.7 / 34.9   107 / 134               200 / 136
// (few CTAs have to split the keys, which paged_attn does at a finer grain).  With heads of 256,
// 4 of them, a CTA here holds 128 rows and one tile, which only the many rows of a batch repay:
//   keys   1 sequence, 96 rows   256 rows      32 sequences, 32 rows   64 rows
//   1024   20.2 / 28.8           24.2 / 32.1   52.7 / 52.0             93.8 / 52.7
//   4096   28.6 / 32.8           46.0 / 46.9   143 / 169               270 / 172
int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  const bool many = int64_t(a.c.batch) * a.c.kv_heads * 2 >= device_sms(dev);
  const int few = many ? 32 : a.c.head_dim == 256 ? 256 : 96;
  if (int64_t(a.c.max_q) * a.group <= few) return launch_paged_attn(a, INT32_MAX, st);
  if (!a.c.cu_q) return launch_paged_prompt(a, 0, st);
  const int status = launch_paged_attn(a, few, st);
  return status != SPECTRA_OK ? status : launch_paged_prompt(a, few, st);
}

int paged_prompt_timeouts(long long* out, bool reset) { return read_timeout_counter(g_paged_prompt_timeouts, out, reset); }

}  // namespace spectra
