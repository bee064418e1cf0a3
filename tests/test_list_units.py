"""csrc/list_units.h, which units of its listed blocks a row of the attention
reads, run on the host over lists, windows and positions: every key that the
row sees lies in one of them, the first and the last hold such a key, and the
pieces of a split row are all of them, each once."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "spectra_b200" / "csrc"

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "list_units.h"

using namespace spectra;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (block %d, lo %d, hi %d, list %x)\n", __LINE__, #x, 1 << bl, lo, hi, list); std::exit(1); } } while (0)

int main() {
  const int ul = 5;
  for (int bl = 5; bl <= 9; bl += 2)
    for (unsigned list = 0; list < 32; ++list)  // blocks of a sequence of up to 5
      for (int hi = 0; hi <= 5 << bl; hi += hi % 32 == 0 || hi % 32 == 31 ? 1 : 15)
        for (int lo = 0; lo <= hi + 40; lo += lo % 32 == 0 || lo % 32 == 31 ? 1 : 30) {
          std::vector<int> kept;  // as the kernel keeps them
          for (int e = 0; e < 5; ++e)
            if (list >> e & 1u && e <= (hi - 1) >> bl && e >= lo >> bl) kept.push_back(e);
          const int n = int(kept.size());
          const UnitRange r = list_units(n, n ? kept[0] : 0, n ? kept[n - 1] : 0, lo, hi, bl, ul);
          CHECK(0 <= r.begin && r.begin <= r.end && r.end <= n << (bl - ul));
          auto first_of = [&](int u) { return (kept[u >> (bl - ul)] << bl) + ((u & ((1 << (bl - ul)) - 1)) << ul); };
          auto seen = [&](int u) { return first_of(u) < hi && first_of(u) + (1 << ul) > lo && lo < hi; };
          for (int u = 0; u < n << (bl - ul); ++u) CHECK(!seen(u) || (r.begin <= u && u < r.end));
          if (lo < hi && r.begin < r.end) CHECK(seen(r.begin) && seen(r.end - 1));
          CHECK(r.end - r.begin <= most_list_units(n, hi, bl, ul));
          for (int pieces = 1; pieces <= 7; ++pieces) {
            int at = r.begin;
            for (int p = 0; p < pieces; ++p) {
              const UnitRange m = piece_of(r, p, pieces);
              CHECK(m.begin == at && m.end >= at);
              at = m.end;
            }
            CHECK(at == r.end);
          }
        }
  const int bl = 16, lo = 0, hi = 100;
  const unsigned list = 1;
  CHECK(list_units(1, 0, 0, lo, hi, bl, ul).end == 4 && most_list_units(1, 100, bl, ul) == 4);
  // positions near the end of what 32 bits count
  const int last = (1 << 15) - 1, far = 2147483647;
  const UnitRange r = list_units(1, last, last, far - 70, far, bl, ul);
  CHECK(r.begin == 2048 - 3 && r.end == 2048);
  CHECK(most_list_units(1024, far, bl, ul) == 1024 * 2048);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_the_units_that_a_row_reads(tmp_path):
    src, exe = tmp_path / "list_units.cpp", tmp_path / "list_units"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-I", str(CSRC), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
