"""Waits of the paged attention kernels that may give up: their result decides
where a warp goes, so all of its lanes have to get the same one.  (Read from
the source: a wait that runs out cannot be staged in these kernels.)"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "spectra_b200" / "csrc"


@pytest.mark.parametrize("name", ["paged_attn.cu", "paged_prompt.cu"])
def test_a_wait_whose_result_is_used_is_voted_on(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    uses = list(re.finditer(r"(?:sm100::)?\bmbar_wait(?:_inline|_poll|_slow)?\(", text))
    assert uses
    for m in uses:
        before = text[:m.start()].rstrip()
        voted = before.endswith("__all_sync(0xffffffffu,")
        # a statement of its own: waited for, whatever comes of it
        unused = before[-1] in ";{}" or before.endswith(")") and re.search(r"\bif \([^;{}]*\)$", before)
        assert voted or unused, text[m.start() - 80:m.end() + 60]
