// Internal interface of the logit rules (not part of the public C ABI; the
// extern "C" wrapper lives in abi.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "spectra_b200.h"

namespace spectra {

struct LogitArgs {
  SpectraLogitRules r;
  const void* x; int x_dtype; int64_t x_rs;       // [M, N]
  void* out; int out_dtype; int64_t out_rs;       // [M, N] or NULL
  int64_t* idx; float* val;                       // [M] or NULL
  int64_t M, N, idx_offset;
  uint2* tops;                                    // [M][parts of a row]: the workspace
};
// `r` as the kernels see it: max_ids and n_bias 0 where a rule is left out.
size_t logits_workspace_bytes(const SpectraLogitRules& r, int64_t M, int64_t N, int x_dtype, bool tokens);
int launch_logits(const LogitArgs& a, cudaStream_t st);

}  // namespace spectra
