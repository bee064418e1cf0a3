// Rules on a step's logits and the greedy choice under them, for sm_100a.
//
// For token v of row m, in fp32, every step rounded by itself:
//   v in ids[0 .. len):  x = x > 0 ? x / r : x r
//   n = times of v in ids[prompt .. len), n > 0:  x = (x - f n) - p
//   x = x + b(v),  b of the last entry that names v
//   v not allowed:  x = -inf
// and the token: first maximum of x among the allowed (NaN above every number).
//
// A row belongs to a cluster of 8 CTAs, each a slice of the vocabulary in
// chunks.  A chunk has a word of shared memory per token: 19 bits count the
// token's ids, one says that the prompt holds it, 12 name its bias.  Whole
// numbers are added up (atomics in shared memory), so their order does not
// matter, and a list of any length costs one pass over it whatever the
// vocabulary.  Most words stay 0: their logits go through untouched.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "gemv_mma.cuh"
#include "logits.h"
#include "sm100_ptx.cuh"

namespace spectra {

namespace {

constexpr int kThreads = 512;
constexpr int kCluster = 8;                     // CTAs per row (a portable cluster size)
constexpr int kUnits = 4;                       // of 8 columns, that a thread takes in a chunk
constexpr int kChunk = kThreads * kUnits * 8;   // columns
constexpr uint32_t kCountBits = 19, kPrompt = 1u << kCountBits, kSlot = kCountBits + 1;
constexpr uint32_t kCountMask = kPrompt - 1, kLow = (1u << kSlot) - 1;
static_assert(SPECTRA_MAX_RULE_IDS <= kCountMask && SPECTRA_MAX_RULE_BIASES < (1 << (32 - kSlot)), "a word's fields");

// Larger value first, a NaN above every number, the lower index among equals; index -1: none.
__device__ __forceinline__ bool better(float v, int64_t i, float bv, int64_t bi) {
  if (i < 0 || bi < 0) return i >= 0;
  const bool vn = v != v, bn = bv != bv;
  if (vn || bn) return vn && (!bn || i < bi);
  return v > bv || (v == bv && i < bi);
}

__device__ __forceinline__ int clamp_len(int v, int64_t most) { return v < 0 ? 0 : (v < most ? v : int(most)); }

__global__ void __launch_bounds__(kThreads) logits_kernel(LogitArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint32_t words[];  // [kChunk]
  sm100::pdl_wait();
  const int64_t m = blockIdx.y;
  const SpectraLogitRules& r = a.r;
  const int64_t lo = min(a.N, int64_t(cluster.block_rank()) * a.span), hi = min(a.N, lo + a.span);
  const int len = !r.ids ? 0 : (r.lengths ? clamp_len(r.lengths[m], r.max_ids) : int(r.max_ids));
  const int prompt = r.prompt_lengths ? clamp_len(r.prompt_lengths[m], len) : 0;
  const float rep = r.repetition ? r.repetition[m] : 1.f;
  const float freq = r.frequency ? r.frequency[m] : 0.f, pres = r.presence ? r.presence[m] : 0.f;
  float bv = -INFINITY;
  int64_t bi = -1;
  for (int64_t c0 = lo; c0 < hi; c0 += kChunk) {
    const int n = int(min(hi - c0, int64_t(kChunk)));
    const int64_t token0 = c0 + a.idx_offset;
    if (len > 0 || r.n_bias > 0) {
      for (int i = threadIdx.x; i < n; i += kThreads) words[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const int64_t at = int64_t(r.ids[m * r.ids_stride + i]) - token0;
        if (at < 0 || at >= n) continue;
        if (i < prompt)
          atomicOr(words + at, kPrompt);
        else
          atomicAdd(words + at, 1u);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < r.n_bias; i += kThreads) {
        const int64_t id = r.bias_ids[m * r.bias_ids_stride + i], at = id - token0;
        if (id < 0 || at < 0 || at >= n) continue;
        // (the low bits are settled, so the larger word is the later entry)
        atomicMax(words + at, (words[at] & kLow) | uint32_t(i + 1) << kSlot);
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      float x = load_as_float_cg(a.x, m * a.x_rs + c0 + i, a.x_dtype);
      const uint32_t w = len > 0 || r.n_bias > 0 ? words[i] : 0;
      const uint32_t times = w & kCountMask;
      if (w & (kPrompt | kCountMask)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(times))), pres);
      if (w >> kSlot) x = __fadd_rn(x, r.bias[m * r.bias_stride + (w >> kSlot) - 1]);
      bool ok = true;
      if (r.allowed) {
        const int64_t t = token0 + i;
        ok = (uint32_t(r.allowed[m * r.allowed_stride + (t >> 5)]) >> (t & 31)) & 1u;
        if (!ok) x = -INFINITY;
      }
      if (a.out) store_from_float(a.out, m * a.out_rs + c0 + i, a.out_dtype, x);
      if (ok && better(x, c0 + i, bv, bi)) {
        bv = x;
        bi = c0 + i;
      }
    }
    __syncthreads();
  }
  if (!a.idx) return;  // (the same for every CTA)
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int64_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (better(ov, oi, bv, bi)) {
      bv = ov;
      bi = oi;
    }
  }
  __shared__ float sv[kThreads / 32];
  __shared__ int64_t si[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    sv[warp] = bv;
    si[warp] = bi;
  }
  cluster.sync();
  if (cluster.block_rank() == 0 && warp == 0) {
    bv = -INFINITY;
    bi = -1;
    for (int k = lane; k < kCluster * (kThreads / 32); k += 32) {
      const int cta = k / (kThreads / 32), of = k % (kThreads / 32);
      const float ov = *cluster.map_shared_rank(&sv[of], cta);
      const int64_t oi = *cluster.map_shared_rank(&si[of], cta);
      if (better(ov, oi, bv, bi)) {
        bv = ov;
        bi = oi;
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int64_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (better(ov, oi, bv, bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if (lane == 0) {
      a.idx[m] = bi < 0 ? -1 : bi + a.idx_offset;
      if (a.val) a.val[m] = bv;
    }
  }
  cluster.sync();  // no CTA leaves while the first may still read its shared memory
}

}  // namespace

int launch_logits(LogitArgs a, cudaStream_t st) {
  if (a.M == 0) return SPECTRA_OK;
  if (a.M > 65535) return SPECTRA_ERR_SHAPE;  // grid y
  static PerContextOnce once;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  const int smem = kChunk * int(sizeof(uint32_t));
  e = once.run(dev, [&] { return cudaFuncSetAttribute(logits_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (e != cudaSuccess) return cuda_status(e);
  a.span = (a.N + kCluster - 1) / kCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster, unsigned(a.M));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, logits_kernel, a));
}

}  // namespace spectra
