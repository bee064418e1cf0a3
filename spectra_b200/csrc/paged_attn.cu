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
// Products (mma.sync m16n8k16, fp16 in, fp32 out; with 1-16 rows per head the
// tcgen05 shapes would be mostly padding, and the kernel is bound by bytes
// and by unpacking instructions, not by the tensor pipe):
//   S^T = K Q^T: A = raw key codes, 16 tokens x 16 features.  A nibble under
//     fp16's 0x6400 is 1024 + q where it lies in bits 0-3 and 1024 + 16 q in
//     bits 4-7 (no shift; those queries are divided by 16 and see 64 + q).  With X
//     a group's sum of queries and Y that of its divided ones, the accumulator
//     starts at 960 Y and ends at D = (sum of code times query) + 1024 X; the
//     group's share of t is s (D - (1024 + z) X) in fp32, with 1024 + z again a
//     nibble under 0x6400: the keys are never rounded.
//   O^T = V^T P^T: A = values (q - z) s in fp16 (exact difference, one
//     rounding of the product, 11 bits), B = P in fp16, transposed in
//     registers (movmatrix).  P <= 2^(kLazy + kShift), so fp16 holds it; its rounding
//     (2^-12) averages over the keys, and weights below 2^-28 of the largest are
//     lost from O (not from their sum).  fp16 results are 3.2e-4 off, 2.1e-4 of it
//     their own rounding; values as two exact operands took 18 % longer.
// Queries of both types are scaled per row by a power of two to fp16's upper
// range (exact down to 2^-24 of the row's largest entry).
// The running maximum is only raised when a score passes it by more than
// kLazy (in powers of two): most tiles need no cross-lane reduction and no
// rescaling of O.
//
// Work: a segment is (sequence, key/value head, row tile); a unit is 32
// consecutive tokens of a segment.  The units of all segments, laid end to
// end, are dealt to the CTAs in equal contiguous shares, whatever the lengths
// of the sequences; a segment that several CTAs share is put together by the
// last of them to finish, always in the same order.
//
// Lists (attention over some blocks of the keys): a segment is one token of one
// key/value head, its units are those of the blocks listed for it, from the first
// to the last key that the token sees (list_units.h).  A CTA has a segment, or a
// piece of one where there are few; it first brings the list into order (entries
// above all before them, that hold a key the token sees).
// Measured: 512 segments of 2048 keys, 64 query heads on 8, heads of 128, 46 us
// (3.5 TB/s); 4096 segments of 1024 keys (512 tokens of a prompt) 159 us; one
// token, 2048 keys, 9.4 us.  Bound like the rest by unpacking: 430 instructions a
// tile of 16 tokens, issue slots 67 % taken, and every token unpacks its own blocks.
//
// Measured: one token over 131072, 32 query heads on 8, heads of 128, 49.6
// us (3.2 TB/s); one token of 64 ragged sequences up to 8192, 64 on 8, 102 us
// (3.6 TB/s); one over 1024 9.2 us, nearly all of it launch and latency.  Long
// caches are bound by the unpacking instructions (396 a tile of 16 tokens, a
// third of them for scales and zero points; issue slots 62 % taken, ALU 44 %).
#include <math.h>

#include <algorithm>

#include "copy_ring.h"
#include "gemv_mma.cuh"
#include "list_units.h"
#include "paged_view.cuh"
#include "sm100_ptx.cuh"

namespace spectra {

__device__ int g_paged_attn_timeouts = 0;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnitLog2 = 5;
constexpr int kUnit = 1 << kUnitLog2;  // tokens of a unit: two tiles
constexpr int kStages = 2;         // units in flight per warp
constexpr int kMaxCtas = int(kPagedCounterBytes / sizeof(int));

struct AttnParams {
  PagedAttnArgs a;
  int* counters;
  float* partials;
  int min_share;                   // units a CTA takes at least
  int max_rows;                    // a sequence with more rows per head is the other kernel's
  int segments, pieces;            // lists: all segments, and CTAs per segment
};

// ------------------------------------------------------------ the batch
struct Span {  // a sequence's rows and the keys its rows look at
  int64_t first;  // first new token
  int count;      // new tokens, up to max_q
  int extra;      // new tokens past max_q
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
  new_rows(a.c, b, s.first, s.count, s.extra);
  const int len = a.c.seq_lens[b];
  s.pos0 = len - s.count - s.extra;
  s.len = len < 0 ? 0 : (len < a.c.limit ? len : a.c.limit);
  s.tiles = s.count * a.group > p.max_rows ? 0 : (s.count * a.group + ROWS - 1) / ROWS;
  s.unit0 = first_key(s.pos0, a.window) / kUnit;
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
  static constexpr int kJoin = ROWS * 66 * 4;                 // weights of 64 parts
  static constexpr int kBig = kRing > kMerge ? (kRing > kJoin ? kRing : kJoin) : (kMerge > kJoin ? kMerge : kJoin);
  static constexpr int kQ = G * NT * 32 * 16;                 // query fragments
  static constexpr int kX = G * NT * 4 * 32;                  // {C, C', C, C'} and {X, X'} of a lane's two rows
  static constexpr int kMeta = ROWS * 16;                     // hi, lo, slope, position of a row
  static constexpr int kCtas = G * NT <= 4 ? 4 : 2;  // per SM: what the registers allow
  // the same for lists where the GPU holds all segments at once so (heads of 128 gain nothing by it)
  static constexpr int kFewListCtas = kCtas == 4 && G < 3 ? 3 : kCtas;
  static constexpr int kSmem = kBig + kQ + kX + kMeta + ROWS * 4 + kWarps * kStages * 8;
  static constexpr int kPartial = ROWS * (D + 2);             // floats of one CTA's partial result
};

// ------------------------------------------------------------ the kernel
// MOD: 0 plain scores, 1 a bias or a cap of up to kLowCap, 2 a higher cap (in MOD 1 its code took
// 35.4 us where 34.2 are taken without it: verification with a bias)
// LISTS 1 and 2: a segment is one token and the blocks listed for it.  2 is for fp16 results: weights as two
// operands, the second what the rounding of the first left (results 2.75e-4 off, 2.1e-4 of it their own rounding;
// 3.2e-4 with one; 5 % longer, and as much for bf16 results where the kernel was the same).
template <int G, int NT, int MOD, int LISTS, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) paged_attn_kernel(AttnParams p) {
  using C = Cfg<G, NT>;
  constexpr int D = C::D, ROWS = C::ROWS;
  constexpr bool SEL = LISTS > 0;
  constexpr TileLayout L{G};
  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;

  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem);
  uint4* qfrag = reinterpret_cast<uint4*>(smem + C::kBig);
  float4* xs = reinterpret_cast<float4*>(smem + C::kBig + C::kQ);
  int4* meta = reinterpret_cast<int4*>(smem + C::kBig + C::kQ + C::kX);
  float* factor = reinterpret_cast<float*>(smem + C::kBig + C::kQ + C::kX + C::kMeta);  // of a row's scores
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBig + C::kQ + C::kX + C::kMeta + ROWS * 4);
  __shared__ long long s_scan[kWarps];
  __shared__ long long s_base;
  __shared__ int s_seq, s_last;
  __shared__ volatile int s_stop;     // a copy did not arrive: the segments after this one load nothing
  __shared__ int s_held[kWarps * kStages];  // tiles of a stage that a page holds
  __shared__ int s_list[SEL ? SPECTRA_MAX_LISTED_BLOCKS : 1];  // blocks that the segment's token sees
  __shared__ int s_tops[2][kWarps], s_kepts[2][kWarps];  // by turns: a turn's are read while the next is under way
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
  sm100::pdl_trigger();

  // ---- this CTA's share of the units (lists: of the segments)
  long long share = 0, begin = 0, end = 0, seq_base = 0;
  int b = -1;
  if constexpr (!SEL) {
    bool over = false;  // a sequence has more new tokens than max_q
    auto units_of = [&](int i) -> long long {
      if (i >= c.batch) return 0;
      const Span s = span_of<ROWS>(p, i);
      over = over || s.extra > 0;
      return (long long)(s.units) * s.tiles * c.kv_heads;
    };
    const long long first_units = units_of(tid);  // (the only ones of a batch of up to kThreads)
    long long total = first_units;
    for (int b0 = kThreads; b0 < c.batch; b0 += kThreads) total += units_of(b0 + tid);
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) s_scan[warp] = total;
    over = __syncthreads_or(over);
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += s_scan[w];
    const long long up = total + gridDim.x - 1;
    share = up < (1ll << 32) ? (long long)(unsigned(up) / gridDim.x) : up / gridDim.x;
    if (share < p.min_share) share = p.min_share;
    begin = share * blockIdx.x;
    end = begin + share < total ? begin + share : total;

    // rows that belong to no sequence, or lie past max_q
    if (c.cu_q) {
      const int64_t row_words = int64_t(a.q_heads) * D;
      auto clear = [&](int64_t t) {
        for (int64_t i = tid; i < row_words; i += kThreads)
          reinterpret_cast<uint16_t*>(a.out)[t * a.o_ts + (i / D) * a.o_hs + i % D] = 0;
      };
      const int held = c.cu_q[c.batch];
      for (int64_t t = (held < 0 ? 0 : held) + int64_t(blockIdx.x); t < c.total; t += gridDim.x) clear(t);
      if (over) {
        for (int i = blockIdx.x; i < c.batch; i += gridDim.x) {
          const Span s = span_of<ROWS>(p, i);
          for (int64_t t = s.first + s.count; t < s.first + s.count + s.extra; ++t) clear(t);
        }
      }
    }
    if (begin >= end) return;

    // ---- the sequence where the share begins
    long long base = 0;
    for (int b0 = 0; b0 < c.batch; b0 += kThreads) {
      const long long mine = b0 == 0 ? first_units : units_of(b0 + tid);
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
    b = s_seq;
    seq_base = s_base;
    if (b < 0) return;
  }

  const bool bf16 = a.dtype == SPECTRA_DT_BF16;
  const int per_page = 1 << (c.page_log2 - 4);  // tiles
  CopyRing<kStages> ring_order;
  const uint32_t magic = fp16_1024();
  long long at = begin;
  int work = int(blockIdx.x);  // lists: piece of a segment

  while (SEL ? work < p.segments * p.pieces : at < end) {
    const int segment = SEL ? work / p.pieces : 0, piece = SEL ? work - segment * p.pieces : 0;
    Span s;
    long long seg_begin = 0, seg_end = 0;
    int head, row0, u_begin, u_stop, u_end, rows;
    const int of_token = (a.group + ROWS - 1) / ROWS;
    if constexpr (SEL) {
      // ---- a segment: token, key/value head, row tile; neighbours share a token
      const int t = segment / (c.kv_heads * of_token), rest = segment - t * (c.kv_heads * of_token);
      head = rest / of_token;
      row0 = (rest - head * of_token) * ROWS;
      rows = min(ROWS, a.group - row0);
      b = sequence_of(c, t);
      s = Span{t, 1, 0, 0, -1, 0, 1, 1};  // a row of no sequence, or past max_q: no keys
      if (b >= 0) {
        int64_t first;
        int count, extra;
        new_rows(c, b, first, count, extra);
        const int len = c.seq_lens[b], of_seq = int(t - first);
        if (of_seq < count) {
          s.pos0 = len - count - extra + of_seq;
          s.len = len < 0 ? 0 : (len < c.limit ? len : c.limit);
        }
      }
      // the token's list: entries above all before them that hold a key it sees
      const int pos = s.pos0, hi = pos < 0 ? 0 : (a.causal ? min(s.len, pos + 1) : s.len);
      const int lo = first_key(pos, a.window);
      const int* list = a.blocks + t * a.b_ts + head * a.b_hs;
      int most = -1, kept = 0;  // of the entries before
      for (int i0 = 0; i0 < a.count; i0 += kThreads) {
        const int e = i0 + tid < a.count ? list[i0 + tid] : -1;
        int* s_top = s_tops[i0 / kThreads & 1];
        int* s_kept = s_kepts[i0 / kThreads & 1];
        int top = e;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, top, o);
          if (lane >= o) top = max(top, up);
        }
        if (lane == 31) s_top[warp] = top;
        top = __shfl_up_sync(0xffffffffu, top, 1);
        if (lane == 0) top = -1;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) top = max(top, s_top[w]);
        }
        const bool ok = e > max(top, most) && e <= (hi - 1) >> a.block_log2 && e >= lo >> a.block_log2;
        const uint32_t oks = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_kept[warp] = __popc(oks);
        __syncthreads();
        int slot = kept + __popc(oks & ((1u << lane) - 1));
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) slot += s_kept[w];
          kept += s_kept[w];
          most = max(most, s_top[w]);
        }
        if (ok) s_list[slot] = e;
      }
      __syncthreads();
      // (a block may be far larger than what the row sees of it: 512 segments of 100 keys in blocks of 65536
      // took 1.27 ms as whole blocks, as long as in blocks of 128 this way)
      const UnitRange seen = list_units(kept, s_list[0], s_list[kept > 0 ? kept - 1 : 0], lo, hi, a.block_log2, kUnitLog2);
      const UnitRange mine = piece_of(seen, piece, p.pieces);
      u_begin = mine.begin;
      u_stop = mine.end;
      u_end = s_stop ? u_begin : u_stop;
    } else {
      // ---- the segment that holds unit `at`
      s = span_of<ROWS>(p, b);
      long long seq_units = (long long)(s.units) * s.tiles * c.kv_heads;
      while (at >= seq_base + seq_units) {
        seq_base += seq_units;
        ++b;
        s = span_of<ROWS>(p, b);
        seq_units = (long long)(s.units) * s.tiles * c.kv_heads;
      }
      const int seg = int(unsigned(at - seq_base) / unsigned(s.units));  // (the launch checks that a sequence's fit)
      seg_begin = seq_base + (long long)(seg) * s.units;
      seg_end = seg_begin + s.units;
      head = seg / s.tiles;
      row0 = (seg - head * s.tiles) * ROWS;
      u_begin = s.unit0 + int(at - seg_begin);
      u_stop = s.unit0 + int((seg_end < end ? seg_end : end) - seg_begin);
      // nothing held, or a copy that did not arrive in an earlier segment: nothing to load.  (After a
      // loss the results are undefined, but every segment is counted, so that the counters end at zero.)
      u_end = s.len > 0 && !s_stop ? u_stop : u_begin;
      rows = min(ROWS, s.count * a.group - row0);
    }
    auto place = [&](int row, int& tok, int& h) {  // token and query head of a row
      if constexpr (SEL) {
        tok = 0;
        h = head * a.group + row0 + row;
      } else {
        tok = (row0 + row) / a.group;
        h = head * a.group + (row0 + row) - tok * a.group;
      }
    };
    auto unit_pos = [&](int u) {  // position of a unit's first token
      if constexpr (SEL) {
        const int of_block = a.block_log2 - kUnitLog2;
        return (s_list[u >> of_block] << a.block_log2) + ((u & ((1 << of_block) - 1)) << kUnitLog2);
      } else {
        return u * kUnit;
      }
    };

    // ---- units to load: warp w takes u_end - 1 - w, - kWarps, ... (the last keys first: a
    // bias on distance only falls on the way).  Lane j knows where the j-th of the next 32
    // of them lies, and in the address's low bits which of its tiles a page holds; where
    // none does, page 0's tile takes its place (the keys are masked, the values finite).
    const int next = u_end - 1 - warp;
    const uint8_t* head_pool = c.pool + int64_t(head) * per_page * C::kTile;
    const int* table = c.tables + b * c.table_stride;
    const bool small = c.page_log2 == 4;  // a page is one tile
    uint64_t here = 0, here1 = 0, ahead = 0, ahead1 = 0;
    auto look = [&](int from, uint64_t& w0, uint64_t& w1) {  // of the warp's units from `from` on
      const int u = next - (from + lane) * kWarps, pos = u >= u_begin ? unit_pos(u) : 0;
      const bool in = u >= u_begin && pos < s.len;
      const int p0 = in ? table[pos >> c.page_log2] : -1;
      const bool h0 = unsigned(p0) < unsigned(c.num_pages);
      w0 = reinterpret_cast<uint64_t>(head_pool + (h0 ? p0 : 0) * c.page_stride + ((pos >> 4) & (per_page - 1)) * C::kTile) + (h0 ? 3 : 0);
      if (small) {
        const int p1 = in && pos + kTileTokens < s.len ? table[(pos >> 4) + 1] : -1;
        const bool h1 = unsigned(p1) < unsigned(c.num_pages);
        w0 -= h0 && !h1 ? 2 : 0;
        w0 += h1 && !h0 ? 2 : 0;
        w1 = reinterpret_cast<uint64_t>(head_pool + (h1 ? p1 : 0) * c.page_stride);
      }
    };
    auto issue = [&](int k, int stage) {  // the warp's k-th unit
      const uint64_t w0 = __shfl_sync(0xffffffffu, here, k & 31);
      const uint64_t w1 = small ? __shfl_sync(0xffffffffu, here1, k & 31) : 0;
      if (lane == 0) {
        uint64_t* bar = bars + warp * kStages + stage;
        uint8_t* dst = ring + (warp * kStages + stage) * C::kStage;
        s_held[warp * kStages + stage] = int(w0) & 3;
        sm100::mbar_arrive_expect_tx(bar, C::kStage);
        const uint8_t* src = reinterpret_cast<const uint8_t*>(w0 & ~uint64_t(15));
        bulk_g2s(dst, src, small ? C::kTile : C::kStage, bar);
        if (small) bulk_g2s(dst + C::kTile, reinterpret_cast<const uint8_t*>(w1), C::kTile, bar);
      }
      if ((k & 31) == 31) {
        here = ahead;
        here1 = ahead1;
        look(k + 33, ahead, ahead1);
      }
    };
    look(0, here, here1);
    if (next - 32 * kWarps >= u_begin) look(32, ahead, ahead1);
    ring_order.start(next >= u_begin ? (next - u_begin) / kWarps + 1 : 0, issue);

    // ---- query fragments: the products' B registers and the groups' sums.  Four
    // lanes a row; every warp reads whole rows and prepares some of their groups.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + g;
      uint32_t raw[G][4], top2 = 0;
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[grp][j] = 0;
      if (row < rows) {
        int tok, h;
        place(row, tok, h);
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (s.first + tok) * a.q_ts + h * a.q_hs + cc * 8;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          if (a.vec) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + grp * 32);
            raw[grp][0] = v.x; raw[grp][1] = v.y; raw[grp][2] = v.z; raw[grp][3] = v.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              raw[grp][j] = uint32_t(src[grp * 32 + 2 * j]) | (uint32_t(src[grp * 32 + 2 * j + 1]) << 16);
          }
        }
      }
      // the row's largest entry
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int j = 0; j < 4; ++j) top2 = bf16 ? max_abs2<true>(top2, raw[grp][j]) : max_abs2<false>(top2, raw[grp][j]);
      uint32_t top = max(top2 >> 16, top2 & 0xFFFFu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // to [2^11, 2^12) (an infinity or NaN: left as it is); both factors are normal numbers
      const float most = bf16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half(uint16_t(top)));
      const int top_e = int(__float_as_uint(most) >> 23);
      const int e = min(top_e == 255 ? 0 : 138 - top_e, 100);
      const float f = __uint_as_float(uint32_t(127 + e) << 23);
      if (warp == 0 && cc == 0) factor[row] = a.scale * __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        if (grp % kWarps != warp) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w = raw[grp][j >> 1];
          x[j] = f * (bf16 ? __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16) : half_of(w, j & 1));
        }
        // pairs (0,4) (1,5) (2,6) (3,7): the order in which the code pairs come
        qfrag[(grp * NT + nt) * 32 + lane] = make_uint4(h2_pack(x[0], x[4]), h2_pack(x[1] * 0.0625f, x[5] * 0.0625f),
                                                        h2_pack(x[2], x[6]), h2_pack(x[3] * 0.0625f, x[7] * 0.0625f));
        float even = (x[0] + x[4]) + (x[2] + x[6]), odd = (x[1] + x[5]) + (x[3] + x[7]);
#pragma unroll
        for (int k = 1; k <= 2; k <<= 1) {
          even += __shfl_xor_sync(0xffffffffu, even, k);
          odd += __shfl_xor_sync(0xffffffffu, odd, k);
        }
        // (1024 + q) even + (64 + q) odd - (1024 + z) X, X = even + odd: the constant is 960 odd
        const float start = 960.f * odd, sum = even + odd;
        const float start1 = __shfl_xor_sync(0xffffffffu, start, 4), sum1 = __shfl_xor_sync(0xffffffffu, sum, 4);
        if (cc == 0 && (g & 1) == 0) {
          float4* x4 = xs + ((grp * NT + nt) * 4 + g / 2) * 2;
          x4[0] = make_float4(start, start1, start, start1);
          x4[1] = make_float4(sum, sum1, 0.f, 0.f);
        }
      }
    }
    if (tid < ROWS) {
      int hi = 0, lo = 0, pos = 0;
      float slope = 0.f;
      if (tid < rows) {
        int tok, h;
        place(tid, tok, h);
        pos = s.pos0 + tok;
        if (pos >= 0) hi = a.causal ? min(s.len, pos + 1) : s.len;
        lo = first_key(pos, a.window);
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

    float c_exp[NT][2];  // from a product to a score in powers of two (MOD: done before)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)  // (not 0, which a masked score of -infinity must not meet)
        c_exp[nt][j] = MOD ? 1.f : fmaxf(factor[nt * 8 + 2 * cc + j] * kLog2e, 1e-37f);
    bool loud = false;  // a maximum past kLoud

    auto arrived = [&](int stage, uint32_t parity) {  // (the vote makes the lanes agree)
      const bool ok = __all_sync(0xffffffffu, sm100::mbar_wait(bars + warp * kStages + stage, parity, &s_never));
      if (!ok && lane == 0) atomicAdd(&g_paged_attn_timeouts, 1);
      return ok;
    };
    for (int u = next; ring_order.more(); u -= kWarps) {
      if (!ring_order.take(arrived)) {
        s_stop = 1;
        break;
      }
      const int stage = ring_order.stage;
      const int held = s_held[warp * kStages + stage];
      const uint8_t* buf = ring + (warp * kStages + stage) * C::kStage;

      // ---- scores of 32 tokens: sc[tile][nt][4], tokens g, g + 8, rows 2cc, 2cc + 1
      float sc[2][NT][4];
      {
        uint32_t w0[2][G], w1[2][G], ks0[2][(2 * G + 3) / 4], ks1[2][(2 * G + 3) / 4], kz0[2][(G + 3) / 4], kz1[2][(G + 3) / 4];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          const uint8_t* t = buf + tile * C::kTile;
          lds<4 * G>(t + L.k_codes() + lane * 4 * G, w0[tile]);
          lds<4 * G>(t + L.k_codes() + L.block() + lane * 4 * G, w1[tile]);
          lds<2 * G>(t + L.k_scales() + g * 2 * G, ks0[tile]);
          lds<2 * G>(t + L.k_scales() + (g + 8) * 2 * G, ks1[tile]);
          lds<G>(t + L.k_zeros() + g * G, kz0[tile]);
          lds<G>(t + L.k_zeros() + (g + 8) * G, kz1[tile]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[tile][nt][i] = 0.f;
        }
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 q = qfrag[(grp * NT + nt) * 32 + lane];
            const float4* x4 = xs + ((grp * NT + nt) * 4 + cc) * 2;
            const float2 x = *reinterpret_cast<const float2*>(x4 + 1);
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
              const uint32_t a0 = w0[tile][grp], a1 = w1[tile][grp];
              const float s0 = half_of(ks0[tile][grp >> 1], grp & 1), s1 = half_of(ks1[tile][grp >> 1], grp & 1);
              const uint32_t zz0 = byte_pair(kz0[tile][grp >> 2], (grp >> 1) & 1), zz1 = byte_pair(kz1[tile][grp >> 2], (grp >> 1) & 1);
              const float z0 = half_of(zz0, grp & 1), z1 = half_of(zz1, grp & 1);  // 1024 + zero point
              float d[4];
              mma_f16(d, code_low(a0, magic), code_low(a1, magic), code_high(a0, magic), code_high(a1, magic), q.x, q.y, x4[0]);
              mma_f16(d, code_low(a0 >> 8, magic), code_low(a1 >> 8, magic), code_high(a0 >> 8, magic), code_high(a1 >> 8, magic), q.z, q.w);
              sc[tile][nt][0] = fmaf(s0, fmaf(-z0, x.x, d[0]), sc[tile][nt][0]);
              sc[tile][nt][1] = fmaf(s0, fmaf(-z0, x.y, d[1]), sc[tile][nt][1]);
              sc[tile][nt][2] = fmaf(s1, fmaf(-z1, x.x, d[2]), sc[tile][nt][2]);
              sc[tile][nt][3] = fmaf(s1, fmaf(-z1, x.y, d[3]), sc[tile][nt][3]);
            }
          }
        }
      }

      // ---- cap, bias, mask
      const int n0 = unit_pos(u);
      if constexpr (MOD != 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int4 r = meta[nt * 8 + 2 * cc + j];
            const float scale = factor[nt * 8 + 2 * cc + j], inv = a.softcap > 0.f ? cap_factor(scale, a.softcap) : 0.f;
            const float back = 1.f / inv;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float& v = sc[k >> 1][nt][2 * (k & 1) + j];
              if constexpr (MOD == 2) v = high_cap(v, inv, back);
              const float t = MOD == 1 && a.softcap > 0.f ? a.softcap * tanh_exp(v * inv) : v * scale;
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
          top[nt][j] = fmaxf(fmaxf(sc[0][nt][j], sc[0][nt][2 + j]), fmaxf(sc[1][nt][j], sc[1][nt][2 + j])) * c_exp[nt][j];
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
        if constexpr (MOD == 0) {
          bool any = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) any = any || fabsf(m[nt][0]) > kLoud || fabsf(m[nt][1]) > kLoud;
          loud = __any_sync(0xffffffffu, any);
        }
      }
      float to_exp[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) to_exp[nt][j] = loud ? 1.f : c_exp[nt][j];
      if (loud) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 8; ++i) sc[i >> 2][nt][i & 3] *= c_exp[nt][i & 1];
      }
      uint32_t pb[2][NT][2];  // P^T fragments: rows as columns
      uint32_t pl[2][NT][2];  // what the rounding to pb left
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"(fmaf(sc[tile][nt][i], to_exp[nt][i & 1], kShift - m[nt][i & 1])));
            l[nt][i & 1] += e[i];
          }
          const uint32_t p0 = h2_pack(e[0], e[1]), p1 = h2_pack(e[2], e[3]);
          pb[tile][nt][0] = transpose8x8(p0);
          pb[tile][nt][1] = transpose8x8(p1);
          if constexpr (LISTS == 2) {
            pl[tile][nt][0] = transpose8x8(h2_pack(e[0] - half_of(p0, 0), e[1] - half_of(p0, 1)));
            pl[tile][nt][1] = transpose8x8(h2_pack(e[2] - half_of(p1, 0), e[3] - half_of(p1, 1)));
          }
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
          const uint32_t z0 = byte_pair(vz0[grp >> 1], grp & 1), z1 = byte_pair(vz1[grp >> 1], grp & 1);  // 1024 + zero points
          const uint32_t c0 = h2_sub(0x63806380u, z0), c1 = h2_sub(0x63806380u, z1);  // 960 - (1024 + z)
          uint32_t v0[4], v1[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x0 = w0[grp] >> (8 * j), x1 = w1[grp] >> (8 * j);
            v0[2 * j] = h2_mul(h2_sub(code_low(x0, magic), z0), vs0[grp]);
            v1[2 * j] = h2_mul(h2_sub(code_low(x1, magic), z1), vs1[grp]);
            v0[2 * j + 1] = h2_mul(h2_fma(code_high(x0, magic), 0x2C002C00u, c0), vs0[grp]);  // (1024 + 16 q) / 16 - 64 - z
            v1[2 * j + 1] = h2_mul(h2_fma(code_high(x1, magic), 0x2C002C00u, c1), vs1[grp]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[grp][0][nt], v0[0], v0[1], v1[0], v1[1], pb[tile][nt][0], pb[tile][nt][1]);
            mma_f16(o[grp][1][nt], v0[2], v0[3], v1[2], v1[3], pb[tile][nt][0], pb[tile][nt][1]);
            if constexpr (LISTS == 2) {
              mma_f16(o[grp][0][nt], v0[0], v0[1], v1[0], v1[1], pl[tile][nt][0], pl[tile][nt][1]);
              mma_f16(o[grp][1][nt], v0[2], v0[3], v1[2], v1[3], pl[tile][nt][0], pl[tile][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      ring_order.next(issue);
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

    const bool whole = SEL ? p.pieces == 1 : seg_begin >= begin && seg_end <= end;
    // the CTAs that share this segment
    const unsigned step = unsigned(share < (1ll << 30) ? share : (1ll << 30));
    int cta0 = seg_begin < begin ? int(blockIdx.x - (unsigned(begin - seg_begin) + step - 1) / step) : int(blockIdx.x);
    int cta1 = int(blockIdx.x) + (seg_end > end ? int(unsigned(seg_end - 1 - begin) / step) : 0);
    float* mine = p.partials + int64_t(2 * blockIdx.x + (seg_begin < begin ? 0 : 1)) * C::kPartial;
    if constexpr (SEL) {  // (a counter per segment, a part per piece)
      cta0 = segment;
      cta1 = segment + p.pieces - 1;
      mine = p.partials + int64_t(work) * C::kPartial;
    }
    auto put = [&](int row, int d, float4 v, float sum) {
      int tok, h;
      place(row, tok, h);
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at_out = (s.first + tok) * a.o_ts + h * a.o_hs + d;
      const float x[4] = {v.x, v.y, v.z, v.w};
      if (a.vec) {
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float lo = sum == 0.f ? 0.f : x[2 * j] * f, hi = sum == 0.f ? 0.f : x[2 * j + 1] * f;
          const __nv_bfloat162 b2 = __floats2bfloat162_rn(lo, hi);
          w[j] = bf16 ? *reinterpret_cast<const uint32_t*>(&b2) : h2_pack(lo, hi);
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at_out) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) store_from_float(a.out, at_out + j, a.dtype, sum == 0.f ? 0.f : x[j] * f);
      }
    };
    auto add = [](float4& acc, float f, const float4& v) {
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    };
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
      float top = kNone, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge[w * C::kSlab + row * (D + 4) + D]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* slab = merge + w * C::kSlab + row * (D + 4);
        const float f = exp2f(slab[D] - top);
        sum = fmaf(f, slab[D + 1], sum);
        add(acc, f, *reinterpret_cast<const float4*>(slab + d));
      }
      if (whole) {
        put(row, d, acc, sum);
      } else {
        *reinterpret_cast<float4*>(mine + row * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(mine + ROWS * D + 2 * row) = make_float2(top, sum);
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
        // 64 parts at a time: a warp per row finds their weights, then every thread adds its
        // items up, 16 loads in flight (one after the other took 7 us of a 34 us call).  The first CTA's part is its last segment's (slot 1),
        // the others' their first's (slot 0).
        const float* parts = p.partials + (SEL ? int64_t(segment) * p.pieces : int64_t(2 * cta0)) * C::kPartial;
        const int n = cta1 - cta0 + 1;
        auto part_of = [&](int k) { return parts + int64_t(SEL ? k : k == 0 ? 1 : 2 * k) * C::kPartial; };
        constexpr int kItems = (ROWS * D / 4 + kThreads - 1) / kThreads, kRowsOfWarp = ROWS / kWarps;
        constexpr int kFlight = kItems >= 4 ? 4 : 16 / kItems;  // parts whose loads are in flight
        float* weight = merge;                        // [ROWS][64] (every thread is past its reads of the slabs)
        float* fade = merge + ROWS * 64;              // [ROWS] of what has been added up
        float* whole_sum = merge + ROWS * 65;         // [ROWS]
        float top[kRowsOfWarp], sum[kRowsOfWarp];
        float4 acc[kItems];
#pragma unroll
        for (int j = 0; j < kItems; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kRowsOfWarp; ++j) {
          top[j] = kNone;
          sum[j] = 0.f;
        }
        for (int k0 = 0; k0 < n; k0 += 64) {
          float2 ml[kRowsOfWarp][2];
#pragma unroll
          for (int j = 0; j < kRowsOfWarp; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int k = k0 + 32 * x + lane, row = warp + j * kWarps;
              ml[j][x] = make_float2(kNone, 0.f);
              if (k < n && row < rows) ml[j][x] = __ldcg(reinterpret_cast<const float2*>(part_of(k) + ROWS * D + 2 * row));
            }
#pragma unroll
          for (int j = 0; j < kRowsOfWarp; ++j) {
            const int row = warp + j * kWarps;
            float up = fmaxf(top[j], fmaxf(ml[j][0].x, ml[j][1].x));
#pragma unroll
            for (int k = 16; k; k >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, k));
            const float f = exp2f(top[j] - up), f0 = exp2f(ml[j][0].x - up), f1 = exp2f(ml[j][1].x - up);
            float add_up = f0 * ml[j][0].y + f1 * ml[j][1].y;
#pragma unroll
            for (int k = 16; k; k >>= 1) add_up += __shfl_xor_sync(0xffffffffu, add_up, k);
            top[j] = up;
            sum[j] = fmaf(sum[j], f, add_up);
            weight[row * 64 + lane] = f0;
            weight[row * 64 + 32 + lane] = f1;
            if (lane == 0) {
              fade[row] = f;
              whole_sum[row] = sum[j];
            }
          }
          __syncthreads();
          int row[kItems], d[kItems];
#pragma unroll
          for (int j = 0; j < kItems; ++j) {
            const int i = min(tid + j * kThreads, rows * (D / 4) - 1);
            row[j] = i / (D / 4);
            d[j] = (i - row[j] * (D / 4)) * 4;
            const float f = fade[row[j]];
            acc[j] = make_float4(acc[j].x * f, acc[j].y * f, acc[j].z * f, acc[j].w * f);
          }
          const int most = min(64, n - k0);
          for (int k = 0; k < most; k += kFlight) {  // (past the last part: the last again, with weight 0)
            float4 v[kFlight][kItems];
#pragma unroll
            for (int x = 0; x < kFlight; ++x)
#pragma unroll
              for (int j = 0; j < kItems; ++j)
                v[x][j] = __ldcg(reinterpret_cast<const float4*>(part_of(k0 + min(k + x, most - 1)) + row[j] * D + d[j]));
#pragma unroll
            for (int x = 0; x < kFlight; ++x)
#pragma unroll
              for (int j = 0; j < kItems; ++j) add(acc[j], k + x < most ? weight[row[j] * 64 + k + x] : 0.f, v[x][j]);
          }
          __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
          const int i = tid + j * kThreads, row = i / (D / 4), d = (i - row * (D / 4)) * 4;
          if (i < rows * (D / 4)) put(row, d, acc[j], whole_sum[row]);
        }
      }
    }
    sm100::fence_proxy_async_smem();
    __syncthreads();  // before the ring, the fragments and the row table are written again
    if constexpr (SEL)
      work += gridDim.x;
    else
      at = seg_begin + (u_stop - s.unit0);
  }
}

template <int G, int NT, int MOD, int LISTS, int CTAS>
int launch_one(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  using C = Cfg<G, NT>;
  static PerContextOnce once;
  static int ctas_per_sm[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  auto kern = paged_attn_kernel<G, NT, MOD, LISTS, CTAS>;
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
  const int64_t units = (a.c.limit + kUnit - 1) / kUnit + 1;
  const int64_t of_one = int64_t(a.c.kv_heads) * tiles * units;
  if (!LISTS && of_one >= (int64_t(1) << 30)) return SPECTRA_ERR_SHAPE;
  const int64_t most = a.c.batch * of_one;
  const int64_t room = std::min<int64_t>(int64_t(device_sms(dev)) * std::max(1, ctas_per_sm[dev]), kMaxCtas);
  int64_t parts = 0;
  int64_t grid = std::max<int64_t>(1, std::min<int64_t>(room, (most + p.min_share - 1) / p.min_share));
  if (LISTS) {
    const int64_t segments = a.c.total * a.c.kv_heads * ((a.group + C::ROWS - 1) / C::ROWS);
    if (segments > INT32_MAX - kMaxCtas) return SPECTRA_ERR_SHAPE;
    const int64_t list = most_list_units(a.count, a.c.limit, a.block_log2, kUnitLog2);
    p.segments = int(segments);
    // As many CTAs per segment as the GPU holds; whole ones by turns where there are more segments than CTAs
    // (512 segments of 64 units in 3 pieces each on 444 CTAs: 72.7 us, whole 62.6)
    p.pieces = int(std::max<int64_t>(1, std::min<int64_t>(room / segments, list / p.min_share)));
    grid = std::min<int64_t>(room, segments * p.pieces);
    if (p.pieces > 1) parts = segments * p.pieces;
  }
  p.counters = static_cast<int*>(a.workspace);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kPagedCounterBytes);
  if (!LISTS) parts = 2 * grid;
  if (a.workspace_bytes < kPagedCounterBytes + size_t(parts) * C::kPartial * sizeof(float)) return SPECTRA_ERR_WORKSPACE;

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

template <int G, int NT, int LISTS, int CTAS>
int launch_mod(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  if (a.softcap > kLowCap) return launch_one<G, NT, 2, LISTS, CTAS>(a, max_rows, st);
  return a.softcap > 0.f || a.slopes ? launch_one<G, NT, 1, LISTS, CTAS>(a, max_rows, st)
                                     : launch_one<G, NT, 0, LISTS, CTAS>(a, max_rows, st);
}

// CTAs per SM.  Lists of heads of 32 and 64: three, with more registers, where the GPU holds all segments at once that
// way, four above that.  Measured, 24 blocks of 32, 32 query heads on 8 of 64, with three and with four: 128 segments
// 10.0 and 10.4 us, 384 11.5 and 13.3, 512 19.1 and 13.6, 768 (two turns either way) 21.4 and 22.8, 1024 29.1 and 25.5,
// 4096 98.8 and 88.3; heads of 32: 384 9.5 and 10.6, 512 16.8 and 10.7, 768 17.3 and 18.1, 4096 83.4 and 69.3.  (Heads
// of 128 with three: 512 segments 62.6, with four 45.9.)
template <int G, int NT, int LISTS>
int launch_ctas(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  using C = Cfg<G, NT>;
  if constexpr (LISTS && C::kFewListCtas < C::kCtas) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e);
    const int64_t segments = a.c.total * a.c.kv_heads * ((a.group + C::ROWS - 1) / C::ROWS);
    if (segments <= int64_t(device_sms(dev)) * C::kFewListCtas) return launch_mod<G, NT, LISTS, C::kFewListCtas>(a, max_rows, st);
  }
  return launch_mod<G, NT, LISTS, C::kCtas>(a, max_rows, st);
}

template <int G, int LISTS>
int launch_rows(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  // up to 8 rows per key/value head (lists: of one token): one column tile (fewer registers, more CTAs per SM);
  // heads of 256 have no registers for two
  if (G == 8 || (LISTS ? 1 : int64_t(a.c.max_q)) * a.group <= 8)
    return launch_ctas<G, 1, LISTS>(a, max_rows, st);
  return launch_ctas<G, G == 8 ? 1 : 2, LISTS>(a, max_rows, st);
}

template <int LISTS>
int launch_dim(const PagedAttnArgs& a, int max_rows, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 32: return launch_rows<1, LISTS>(a, max_rows, st);
    case 64: return launch_rows<2, LISTS>(a, max_rows, st);
    case 96: return launch_rows<3, LISTS>(a, max_rows, st);
    case 128: return launch_rows<4, LISTS>(a, max_rows, st);
    case 256: return launch_rows<8, LISTS>(a, max_rows, st);
  }
  return SPECTRA_ERR_UNSUPPORTED;
}

}  // namespace

int launch_paged_attn(const PagedAttnArgs& a, int max_rows, cudaStream_t st) { return launch_dim<0>(a, max_rows, st); }
int launch_paged_attn_blocks(const PagedAttnArgs& a, cudaStream_t st) {
  return a.dtype == SPECTRA_DT_BF16 ? launch_dim<1>(a, INT32_MAX, st) : launch_dim<2>(a, INT32_MAX, st);
}

size_t paged_attn_workspace_bytes(int head_dim) {
  return kPagedCounterBytes + size_t(kMaxCtas) * 2 * 16 * (head_dim + 2) * sizeof(float);
}

int paged_attn_timeouts(long long* out, bool reset) { return read_timeout_counter(g_paged_attn_timeouts, out, reset); }

}  // namespace spectra
