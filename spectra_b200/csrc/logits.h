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
};
int launch_logits(LogitArgs a, cudaStream_t st);

}  // namespace spectra
