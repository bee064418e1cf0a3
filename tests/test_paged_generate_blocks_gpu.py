"""examples/paged_generate.py with chosen blocks and penalties: eager and
replayed steps give the same tokens, the tokens are the oracle's choice from the
logits, and a choice of every block is the whole attention."""
import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import logits as R

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "paged_generate.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_generate", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def model_of(example, **kw):
    return example.PagedLlama(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, inner=512, pages=40, page_size=32, **kw)


def prompts_of(*lens):
    g = torch.Generator().manual_seed(2)
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("choose", [0, 3])
def test_replayed_steps_are_the_eager_ones(example, choose):
    model, prompts = model_of(example, choose=choose), prompts_of(5, 330, 1, 96)
    kw = dict(repetition=1.3, presence=0.4)
    a, la = model.generate(prompts, 40, graph=True, **kw)
    b, lb = model.generate(prompts, 40, graph=False, **kw)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_tokens_are_chosen_under_the_penalties(example):
    model, prompts = model_of(example, choose=4), prompts_of(70, 200)
    tokens, logits = model.generate(prompts, 24, repetition=1.5, presence=0.7)
    plain, _ = model.generate(prompts, 24)
    for b, p in enumerate(prompts):
        ids = list(p)
        for i, t in enumerate(tokens[b].tolist()):
            assert R.adjust(logits[b, i].float().cpu().numpy(), ids=ids, prompt=len(p), repetition=1.5, presence=0.7)[1] == t
            ids.append(t)
    assert not torch.equal(plain, tokens)


def test_a_choice_of_every_block_is_the_whole_attention(example):
    prompts = prompts_of(5, 230, 64)
    tokens, logits = model_of(example, choose=9).generate(prompts, 12)
    want, dense = model_of(example).generate(prompts, 12)
    # the first steps on equal tokens; both paths round to bf16 at every linear (2^-8 each)
    same = (tokens == want).long().cumprod(1).bool()
    err = (logits.float() - dense.float()).abs().amax(-1) / dense.float().abs().amax(-1)
    before = torch.cat([torch.ones_like(same[:, :1]), same[:, :-1]], 1)
    assert float(err[before].max()) <= 6e-2
