// The order in which a warp issues and waits for its bulk copies, STAGES of
// them in flight.  Apart from the kernels, so that a host program can run it
// through lost copies.
#pragma once

#include <stdint.h>

#if defined(__CUDACC__)
#define SPECTRA_RING_FN __host__ __device__ __forceinline__
#else
#define SPECTRA_RING_FN inline
#endif

namespace spectra {

// A run takes units 0 .. units - 1; unit k uses stage k % STAGES.  For each
// unit: take(), use its stage, next().  A wait that runs out ends the run:
// what else is in flight is waited for once (bounded like every wait), no
// stage's parity moves and nothing more is issued, in this run or a later one.
template <int STAGES>
struct CopyRing {
  uint32_t parity = 0;  // a bit for each stage; outlives a run, as the barriers do
  int units = 0, unit = 0, stage = 0;
  bool lost = false;

  template <class Issue>  // issue(unit, stage)
  SPECTRA_RING_FN void start(int n, Issue&& issue) {
    units = lost ? 0 : n;
    unit = stage = 0;
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
      if (s < units) issue(s, s);
  }
  SPECTRA_RING_FN bool more() const { return unit < units; }
  template <class Wait>  // wait(stage, parity): whether that phase has completed
  SPECTRA_RING_FN bool take(Wait&& wait) {
    if (wait(stage, (parity >> stage) & 1u)) return true;
    for (int j = 1; j < STAGES && unit + j < units; ++j) {
      const int s = (stage + j) % STAGES;
      wait(s, (parity >> s) & 1u);
    }
    lost = true;
    units = unit;
    return false;
  }
  template <class Issue>
  SPECTRA_RING_FN void next(Issue&& issue) {
    parity ^= 1u << stage;
    if (unit + STAGES < units) issue(unit + STAGES, stage);
    ++unit;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
};

}  // namespace spectra
