"""Rules on logits for more rows than one kernel takes (csrc/logits.cu), against
the oracle: every logit bit for bit, every token; also where the maximum of
every slice of a row is a token that the rules change."""
import numpy as np
import pytest
import torch

from spectra_b200 import kernels as SK
from spectra_b200 import logits as LG
from tests.test_logits_gpu import DEV, DTYPES, Batch, bits, check

pytestmark = pytest.mark.gpu

SHAPES = [  # rows, vocab, ids, biases, mask (two kernels from 297 rows, 149 of more than 16384 or 75 of more than 32768)
    (297, 1, 3, 1, None), (300, 31, 4, 2, 0.5), (301, 515, 64, 3, 0.5), (297, 1000, 0, 5, None), (298, 1001, 300, 17, 0.5),
    (149, 16385, 2000, 64, 0.02), (151, 20003, 5400, 61, 0.99), (150, 20003, 5461, 1, 0.7), (76, 50001, 1200, 40, 0.3),
    (38, 128256, 3000, 100, None), (38, 128256, 0, 0, 0.3), (40, 200003, 700, 9, 0.5), (38, 270001, 50, 3, None),
]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,ids,biases,mask", SHAPES)
def test_all_rules_bit_for_bit(rows, vocab, ids, biases, mask, dt):
    b = Batch(rows, vocab, dt, ids, biases, mask, seed=vocab + rows)
    want, tokens = b.want()
    x = b.x.to(DEV)
    got, chosen = LG.adjust_logits(x, b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()
    assert torch.equal(bits(x), bits(b.x))
    check(LG.adjust_logits(x, b.rules()), want, b.dtype)
    value = np.array([w[t] if t >= 0 else -np.inf for w, t in zip(want, tokens)], np.float32)
    idx, val = SK.argmax(x, with_values=True, rules=b.rules())
    assert idx.tolist() == tokens.tolist() and np.array_equal(val.cpu().numpy(), value)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["repeated", "biased", "not allowed"])
def test_maxima_that_the_rules_take_away(kind, dt):
    vocab, rows = 70001, 40
    b = Batch(rows, vocab, dt, mask=0.9, seed=21)
    top = b.x.float().argsort(-1, descending=True)[:, :2500].to(torch.int32)  # (every slice's highest are among them)
    if kind == "repeated":
        b.kw.update(ids=top, lengths=torch.full((rows,), 2500, dtype=torch.int32), prompt_lengths=torch.zeros(rows, dtype=torch.int32),
                    repetition=torch.full((rows,), 30.0), frequency=torch.zeros(rows), presence=torch.full((rows,), 9.0))
    elif kind == "biased":
        b.kw.update(bias_ids=top, bias=torch.full(top.shape, -50.0))
    else:
        b.allowed.scatter_(1, top.long(), False)
        from tests.test_logits_gpu import pack
        b.kw["allowed"] = pack(b.allowed)
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()


def test_ties_nan_and_rows_without_any_allowed_token():
    b = Batch(80, 40000, "bf16", ids=50, biases=5, mask=0.5, seed=4)
    b.x[0] = 1.0
    b.allowed[1] = False
    b.x[2] = -torch.inf
    for m in range(3):
        b.kw["lengths"][m] = 0
        b.kw["bias_ids"][m] = -1
    b.x[3, b.allowed[3, :40000].nonzero()[-1]] = torch.nan
    b.x[4, (~b.allowed[4, :40000]).nonzero()[:, 0]] = torch.nan
    b.x[5, int(b.kw["ids"][5, 0].clamp(0, 39999))] = torch.nan   # a NaN that is penalised stays one
    b.x[6, 100:] = -torch.inf
    from tests.test_logits_gpu import pack
    b.kw["allowed"] = pack(b.allowed)
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist() and chosen[1] == -1


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("offset,width", [(0, 100), (1, 999), (37, 333), (995, 5)])
def test_a_slice_of_the_vocabulary(offset, width, dt):
    b = Batch(300, 1000, dt, ids=90, biases=30, mask=0.6, seed=7)
    want, tokens = b.want(offset, width)
    x = b.x.to(DEV)[:, offset:offset + width]
    got, chosen = LG.adjust_logits(x, b.rules(), idx_offset=offset, with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("at", [0, 1, 3, 8])
def test_in_place_into_a_wider_buffer_and_to_other_types(at, dt):
    b = Batch(150, 20003, dt, ids=500, biases=9, mask=0.7, seed=8)
    want, tokens = b.want()
    wide = torch.full((150, 20024), 7.0, dtype=b.dtype, device=DEV)
    view = wide[:, at:at + 20003]
    view.copy_(b.x)
    same, chosen = LG.adjust_logits(view, b.rules(), out=view, with_tokens=True)
    assert same is view and chosen.tolist() == tokens.tolist()
    check(view, want, b.dtype)
    assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 20003:] == 7).all())
    wide.fill_(7.0)
    LG.adjust_logits(b.x.to(DEV), b.rules(), out=view)
    check(view, want, b.dtype)
    assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 20003:] == 7).all())
    for other in DTYPES.values():
        check(LG.adjust_logits(b.x.to(DEV), b.rules(), out_dtype=other), want, other)


def test_a_captured_choice_follows_its_inputs_and_two_streams():
    b = Batch(150, 20003, "bf16", ids=700, biases=5, mask=0.5, seed=11)
    x, rules = b.x.to(DEV), b.rules()
    LG.adjust_logits(x, rules, with_tokens=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, chosen = LG.adjust_logits(x, rules, with_tokens=True)
    for seed in (12, 13):
        n = Batch(150, 20003, "bf16", ids=700, biases=5, mask=0.5, seed=seed)
        x.copy_(n.x)
        for k, t in n.kw.items():
            (rules._keep[0].get(k) if rules._keep[0].get(k) is not None else rules._keep[1][k]).copy_(t)
        graph.replay()
        want, tokens = n.want()
        check(got, want, b.dtype)
        assert chosen.tolist() == tokens.tolist()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    res = []
    for _ in range(5):  # the same rules on two streams at once
        with torch.cuda.stream(side):
            res.append(LG.adjust_logits(x, rules, with_tokens=True))
        res.append(LG.adjust_logits(x, rules, with_tokens=True))
    torch.cuda.synchronize()
    for y, t in res:
        check(y, want, b.dtype)
        assert t.tolist() == tokens.tolist()
