// Which units of 2^unit_log2 tokens a row reads of the blocks listed for it.
// Apart from the kernels, so that a host program can run it.
#pragma once

#include <stdint.h>

#if defined(__CUDACC__)
#define SPECTRA_UNITS_FN __host__ __device__ __forceinline__
#else
#define SPECTRA_UNITS_FN inline
#endif

namespace spectra {

struct UnitRange {
  int begin, end;
};

// Of `kept` blocks (ascending, first .. last; the units of all of them are counted end to end) for a row
// that sees the keys lo .. hi - 1: from the unit that holds the first key seen in the first block to the
// one that holds the last in the last.  Every block holds a key below hi; none ends at or before lo.
SPECTRA_UNITS_FN UnitRange list_units(int kept, int first, int last, int lo, int hi, int block_log2, int unit_log2) {
  if (kept <= 0) return {0, 0};
  const int of_block = block_log2 - unit_log2, before = lo - (first << block_log2), held = hi - (last << block_log2);
  const int in_last = held >> block_log2 ? 1 << of_block : (held + (1 << unit_log2) - 1) >> unit_log2;
  const int end = ((kept - 1) << of_block) + in_last, begin = before > 0 ? before >> unit_log2 : 0;
  return {begin < end ? begin : end, end};  // (no key seen: a window that begins at or past hi)
}

// Piece `piece` of `pieces` equal ones.
SPECTRA_UNITS_FN UnitRange piece_of(UnitRange r, int piece, int pieces) {
  const int64_t units = r.end - r.begin;
  return {r.begin + int(units * piece / pieces), r.begin + int(units * (piece + 1) / pieces)};
}

// The most units that a list of `count` blocks has in a sequence of up to `limit` tokens.
SPECTRA_UNITS_FN int64_t most_list_units(int64_t count, int64_t limit, int block_log2, int unit_log2) {
  const int64_t of_lists = count << (block_log2 - unit_log2), of_seq = (limit + (int64_t(1) << unit_log2) - 1) >> unit_log2;
  return of_lists < of_seq ? of_lists : of_seq;
}

}  // namespace spectra
