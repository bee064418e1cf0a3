"""examples/paged_generate.py: lengths past what the model holds."""
import pytest
import torch

from tests.test_paged_generate_gpu import example  # noqa: F401

pytestmark = pytest.mark.gpu


def test_refuses_what_it_cannot_hold_and_frees_its_pages(example, monkeypatch):
    model = example.PagedLlama(layers=1, hidden=256, heads=4, kv_heads=2, head_dim=64, inner=512, pages=12, page_size=32,
                               max_len=128)
    free = sorted(model.free)
    for prompts, tokens in (([[1] * 100], 30), ([[1] * 129], 1), ([], 4), ([[1], []], 4), ([[1]], 0)):
        with pytest.raises(ValueError):
            model.generate(prompts, tokens)
    with pytest.raises(RuntimeError, match="pages"):
        model.generate([[1] * 100] * 4, 8)
    tokens, logits = model.generate([[1] * 100, [2] * 99], 29)  # to the last position
    assert torch.equal(logits.argmax(-1), tokens) and torch.isfinite(logits).all()
    monkeypatch.setattr(model, "logits", lambda hidden: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        model.generate([[1, 2, 3]], 4)
    assert sorted(model.free) == free
