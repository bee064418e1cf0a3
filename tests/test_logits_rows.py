"""More rows than the rules on logits take are refused as such, whatever else a
call lacks (no GPU)."""
import pytest
import torch

from spectra_b200 import _lib as L
from spectra_b200 import logits as LG
from tests.test_logits import MANY, adjust


@pytest.mark.parametrize("kw", [{}, dict(N=20000, x_rs=20000, out_rs=20000, ws=None), dict(MANY, ws_bytes=0)])
def test_the_entry_point_refuses_more_than_65535_rows(kw):
    assert adjust(dict(allowed_words=700), **{**kw, "M": 65536}) == L.ERR_SHAPE


def test_rules_of_more_than_65535_rows_are_refused():
    with pytest.raises(ValueError, match="65535"):
        LG.LogitRules(ids=torch.zeros(1, 3, dtype=torch.int32).expand(65536, 3))
    with pytest.raises(RuntimeError):  # (as many as are taken: refused for being on the CPU)
        LG.LogitRules(ids=torch.zeros(1, 3, dtype=torch.int32).expand(65535, 3))
