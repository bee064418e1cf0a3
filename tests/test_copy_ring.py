"""csrc/copy_ring.h, the order in which a warp of the few-token attention
issues and waits for its copies, run on the host through every pattern of lost
copies: it ends after a bounded number of waits, uses nothing that has not
arrived, leaves nothing in flight that it has not waited for, and issues
nothing after a loss."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "spectra_b200" / "csrc"

MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "copy_ring.h"

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (stages %d, units %d+%d, lost %x)\n", __LINE__, #x, S, n0, n1, lost); std::exit(1); } } while (0)

// An mbarrier's phase: test_wait with parity p is true when the phase of that
// parity is the one before the current.
template <int S>
void run(int n0, int n1, unsigned lost) {
  unsigned done[S] = {};         // phases completed
  bool flying[S] = {}, arrived[S] = {};
  int issued = 0, failed = 0, used = 0;
  bool gone = false;
  spectra::CopyRing<S> ring;
  auto issue = [&](int, int s) {
    CHECK(!gone && !flying[s]);
    flying[s] = true;
    arrived[s] = !((lost >> issued++) & 1u);
    if (arrived[s]) ++done[s];
  };
  auto wait = [&](int s, unsigned p) {
    CHECK(s >= 0 && s < S && flying[s]);  // only for a copy in flight, once
    flying[s] = false;
    const bool ok = (done[s] & 1u) != p;
    CHECK(ok == arrived[s]);              // never the phase of an older copy
    failed += !ok;
    return ok;
  };
  for (int n : {n0, n1}) {
    ring.start(n, issue);
    int k = 0;
    while (ring.more()) {
      if (!ring.take(wait)) {
        gone = true;
        break;
      }
      CHECK(ring.unit == k && arrived[ring.stage]);
      ++used;
      ++k;
      ring.next(issue);
    }
    CHECK(gone || k == n);
    for (bool f : flying) CHECK(!f);
  }
  CHECK(gone == ring.lost && failed <= S && (lost != 0 || used == n0 + n1));
}

template <int S>
void all() {
  for (int n0 = 0; n0 <= 6; ++n0)
    for (int n1 = 0; n1 <= 5; ++n1)
      for (unsigned lost = 0; lost < (1u << (n0 + n1)); ++lost) run<S>(n0, n1, lost);
}

int main() {
  all<1>();
  all<2>();
  all<3>();
  std::puts("ok");
}
"""


def test_every_pattern_of_lost_copies(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "model.cpp").write_text(MODEL)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas", f"-I{CSRC}", "model.cpp", "-o", "model"],
                   check=True, cwd=tmp_path)
    r = subprocess.run([str(tmp_path / "model")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_the_kernel_goes_by_the_ring():
    """No wait or copy of the unit loop beside it."""
    text = (CSRC / "paged_attn.cu").read_text()
    assert "ring_order.take(" in text and "ring_order.next(" in text and "ring_order.start(" in text
    assert text.count("mbar_wait") == 1
