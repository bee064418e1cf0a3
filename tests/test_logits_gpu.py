"""Rules on logits (csrc/logits.cu) against the oracle (oracle/logits.py): every
logit bit for bit (fp32 steps, one rounding at the end), every token."""
import numpy as np
import pytest
import torch

from oracle import logits as R
from spectra_b200 import kernels as SK
from spectra_b200 import logits as LG

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Batch:
    """Random logits and rules, on the device and as the oracle takes them."""

    def __init__(self, rows, vocab, dt="bf16", ids=0, biases=0, mask=None, seed=0, spread=3.0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.vocab, self.dtype = rows, vocab, DTYPES[dt]
        self.x = (torch.randn(rows, vocab, generator=g) * spread).to(self.dtype)
        self.kw = {}
        rint = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, dtype=torch.int32)  # noqa: E731
        pick = lambda *v: torch.tensor(v, dtype=torch.float32)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
        if ids:
            few = max(2, vocab // 5)
            self.kw.update(ids=torch.where(torch.rand(rows, ids, generator=g) < 0.7, rint(0, few, rows, ids),
                                           rint(-2, vocab + 3, rows, ids)),
                           lengths=rint(0, ids + 1, rows), prompt_lengths=rint(0, ids + 1, rows),
                           repetition=pick(1.0, 1.1, 0.8, 1.7), frequency=pick(0.0, 0.3, -0.2), presence=pick(0.0, 0.6))
        if biases:
            self.kw.update(bias_ids=rint(-1, min(vocab, 2 * biases) + 2, rows, biases),
                           bias=torch.randn(rows, biases, generator=g) * 4)
        if mask is not None:
            keep = torch.rand(rows, (vocab + 31) // 32 * 32, generator=g) < mask
            self.allowed = keep
            self.kw["allowed"] = pack(keep)

    def rules(self, **kw):
        return LG.LogitRules(**{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in {**self.kw, **kw}.items()})

    def want(self, offset=0, width=None):
        out, tokens = [], []
        for m in range(self.rows):
            k = self.kw
            kw = {}
            if "ids" in k:
                most = k["ids"].shape[1]
                n = min(max(int(k["lengths"][m]), 0), most) if "lengths" in k else most
                kw.update(ids=k["ids"][m, :n].tolist(), prompt=min(max(int(k["prompt_lengths"][m]), 0), n) if "prompt_lengths" in k else 0,
                          **{p: float(k[p][m]) for p in ("repetition", "frequency", "presence") if p in k})
            if "bias_ids" in k:
                kw["biases"] = list(zip(k["bias_ids"][m].tolist(), k["bias"][m].tolist()))
            if "allowed" in k:
                kw["allowed"] = self.allowed[m].numpy()
            x = self.x[m].float().numpy()
            x, token = R.adjust(x[offset:offset + (width or self.vocab)], offset=offset, **kw)
            out.append(x)
            tokens.append(token)
        return np.stack(out), np.array(tokens)


def pack(keep):
    bits = keep.reshape(keep.shape[0], -1, 32).to(torch.int64) << torch.arange(32)
    return bits.sum(-1).to(torch.int32)  # (wraps into the sign bit)


def bits(t):
    return t.detach().cpu().contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()])


def check(got, want, dtype):
    exact = torch.from_numpy(want).to(dtype)
    same = (bits(got) == bits(exact)) | (torch.isnan(got.cpu()) & torch.isnan(exact))
    assert bool(same.all()), f"{int((~same).sum())} logits differ, first at {tuple(int(i) for i in (~same).nonzero()[0])}"


SHAPES = [  # rows, vocab, ids, biases, mask
    (1, 1, 3, 1, None), (1, 31, 4, 2, 0.5), (2, 33, 40, 0, 0.9), (3, 1000, 0, 5, None), (5, 1001, 300, 17, 0.5),
    (4, 4099, 2000, 64, 0.02), (2, 16384, 5000, 300, 0.99), (3, 50001, 1200, 40, 0.3), (2, 128256, 3000, 100, None),
    (1, 200003, 700, 9, 0.5), (65, 515, 64, 3, 0.5),
]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,ids,biases,mask", SHAPES)
def test_all_rules_bit_for_bit(rows, vocab, ids, biases, mask, dt):
    b = Batch(rows, vocab, dt, ids, biases, mask, seed=vocab + rows)
    want, tokens = b.want()
    x = b.x.to(DEV)
    got, chosen = LG.adjust_logits(x, b.rules() if b.kw else None, with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.dtype == torch.int64 and chosen.tolist() == tokens.tolist()
    assert torch.equal(bits(x), bits(b.x))
    value = np.array([w[t] if t >= 0 else -np.inf for w, t in zip(want, tokens)], np.float32)
    idx, val = SK.argmax(x, with_values=True, rules=b.rules())
    assert idx.tolist() == tokens.tolist() and np.array_equal(val.cpu().numpy(), value)


@pytest.mark.parametrize("kw", [dict(ids=50), dict(biases=9), dict(mask=0.4)])
def test_each_rule_alone_and_rounded_to_other_types(kw):
    b = Batch(7, 777, "f32", seed=5, **kw)
    want, tokens = b.want()
    for dt in DTYPES.values():
        got = LG.adjust_logits(b.x.to(DEV), b.rules(), out_dtype=dt)
        check(got, want, dt)


def test_penalties_as_numbers_and_lists_of_full_length():
    b = Batch(4, 300, "bf16", ids=20, seed=2)
    for k in ("lengths", "prompt_lengths", "frequency"):
        del b.kw[k]
    b.kw.update(repetition=torch.full((4,), 1.25), presence=torch.full((4,), 0.5))
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(repetition=1.25, presence=0.5), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()


def test_penalties_as_numbers_whatever_torchs_default_type_is():
    b = Batch(2, 500, ids=40, seed=6)
    rows = {p: torch.full((2,), v) for p, v in (("repetition", 1.3), ("frequency", 0.3), ("presence", 0.7))}  # fp32
    want, _ = LG.adjust_logits(b.x.to(DEV), b.rules(**rows), with_tokens=True)
    try:
        torch.set_default_dtype(torch.bfloat16)
        rules = b.rules(repetition=1.3, frequency=0.3, presence=0.7)
        got = LG.adjust_logits(b.x.to(DEV), rules)
    finally:
        torch.set_default_dtype(torch.float32)
    assert torch.equal(got, want)


def test_lengths_past_their_lists_are_cut():
    b = Batch(6, 500, "f16", ids=30, seed=3)
    b.kw["lengths"] = torch.tensor([-1, -2**31, 0, 31, 2**31 - 1, 30], dtype=torch.int32)
    b.kw["prompt_lengths"] = torch.tensor([5, 0, 7, -3, 10, 2**31 - 1], dtype=torch.int32)
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()


def test_rows_without_any_allowed_token_and_ties():
    b = Batch(5, 2000, "bf16", mask=0.5, seed=4)
    b.x[0] = 1.0                       # all equal: the first allowed
    b.allowed[1] = False               # nothing allowed
    b.x[2] = -torch.inf                # allowed, but all at the bottom: still the first allowed
    b.x[3, b.allowed[3, :2000].nonzero()[-1]] = torch.nan   # a NaN is the maximum where it is allowed
    b.x[4, (~b.allowed[4, :2000]).nonzero()[:, 0]] = torch.nan  # and -infinity where it is not
    b.kw["allowed"] = pack(b.allowed)
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()
    first = lambda m: int(b.allowed[m].nonzero()[0])  # noqa: E731
    assert chosen.tolist()[:3] == [first(0), -1, first(2)] and not torch.isnan(got[4]).any()


def test_infinities_and_the_types_lowest_values_go_through_the_penalties():
    b = Batch(3, 64, "f16", ids=64, biases=4, seed=6)
    b.x[:, 0:5] = torch.tensor([torch.inf, -torch.inf, torch.nan, -65504.0, 65504.0], dtype=torch.float16)
    b.kw["ids"][:, :5] = torch.arange(5)
    b.kw["lengths"][:] = 64
    want, tokens = b.want()
    got, chosen = LG.adjust_logits(b.x.to(DEV), b.rules(), with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("offset,width", [(0, 100), (1, 999), (37, 333), (64, 512), (995, 5)])
def test_a_slice_of_the_vocabulary(offset, width, dt):
    b = Batch(4, 1000, dt, ids=90, biases=30, mask=0.6, seed=7)
    want, tokens = b.want(offset, width)
    x = b.x.to(DEV)[:, offset:offset + width]  # a view: rows off any 16-byte boundary
    got, chosen = LG.adjust_logits(x, b.rules(), idx_offset=offset, with_tokens=True)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()
    assert SK.argmax(x, idx_offset=offset, rules=b.rules()).tolist() == tokens.tolist()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("at", [0, 1, 3, 8])
def test_in_place_and_into_a_wider_buffer(at, dt):
    b = Batch(5, 1003, dt, ids=50, biases=9, mask=0.7, seed=8)
    want, _ = b.want()
    wide = torch.full((5, 1024), 7.0, dtype=b.dtype, device=DEV)
    view = wide[:, at:at + 1003]
    view.copy_(b.x)
    assert LG.adjust_logits(view, b.rules(), out=view) is view
    check(view, want, b.dtype)
    assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 1003:] == 7).all())
    wide.fill_(7.0)
    LG.adjust_logits(b.x.to(DEV), b.rules(), out=view)
    check(view, want, b.dtype)
    assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 1003:] == 7).all())


def test_strided_rules_and_other_shapes():
    b = Batch(6, 321, "bf16", ids=40, biases=8, mask=0.8, seed=9)
    want, tokens = b.want()
    wide = {}
    for k in ("ids", "bias_ids", "bias", "allowed"):
        t = torch.full((6, b.kw[k].shape[1] + 5), 3, dtype=b.kw[k].dtype, device=DEV)
        t[:, 2:-3] = b.kw[k].to(DEV)
        wide[k] = t[:, 2:-3]
    x = b.x.to(DEV).view(2, 3, 321)
    got, chosen = LG.adjust_logits(x, b.rules(**wide), with_tokens=True)
    assert got.shape == (2, 3, 321) and chosen.shape == (2, 3)
    check(got.view(6, 321), want, b.dtype)
    assert chosen.flatten().tolist() == tokens.tolist()
    one = Batch(1, 321, "bf16", ids=40, seed=10)
    w, t = one.want()
    got, chosen = LG.adjust_logits(one.x[0].to(DEV), one.rules(), with_tokens=True)
    assert got.shape == (321,) and chosen.shape == ()
    check(got[None], w, one.dtype)
    assert int(chosen) == t[0]


def test_a_captured_choice_follows_its_inputs():
    b = Batch(3, 5003, "bf16", ids=70, biases=5, mask=0.5, seed=11)
    x, rules = b.x.to(DEV), b.rules()
    LG.adjust_logits(x, rules, with_tokens=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, chosen = LG.adjust_logits(x, rules, with_tokens=True)
    for seed in (12, 13):
        n = Batch(3, 5003, "bf16", ids=70, biases=5, mask=0.5, seed=seed)
        x.copy_(n.x)
        for k, t in n.kw.items():
            (rules._keep[0].get(k) if rules._keep[0].get(k) is not None else rules._keep[1][k]).copy_(t)
        graph.replay()
        want, tokens = n.want()
        check(got, want, b.dtype)
        assert chosen.tolist() == tokens.tolist()


def test_another_stream_and_no_rows():
    b = Batch(4, 900, "bf16", ids=30, mask=0.5, seed=14)
    want, tokens = b.want()
    x, rules = b.x.to(DEV), b.rules()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, chosen = LG.adjust_logits(x, rules, with_tokens=True)
    torch.cuda.current_stream().wait_stream(side)
    check(got, want, b.dtype)
    assert chosen.tolist() == tokens.tolist()
    none = LG.LogitRules(ids=torch.zeros(0, 3, dtype=torch.int32, device=DEV), repetition=1.2)
    got, chosen = LG.adjust_logits(torch.zeros(0, 9, device=DEV), none, with_tokens=True)
    assert got.shape == (0, 9) and chosen.shape == (0,)


def test_the_greedy_head_takes_rules():
    from spectra_b200 import compress as C

    c = C.compress_linear((torch.randn(512, 256, generator=torch.Generator().manual_seed(1)) * 0.1).to(DEV, torch.float16))
    x = torch.randn(1, 256, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    args = (x, c.packed, c.scales, c.zeros)
    kw = dict(outlier_idx=c.outlier_idx, outlier_w=c.outlier_w, marlin_layout=True)
    tok, logits = SK.lm_head_greedy(*args, **kw)
    banned = torch.full((1, 1), int(tok), dtype=torch.int32, device=DEV)
    rules = LG.LogitRules(bias_ids=banned, bias=torch.full((1, 1), -1e9, device=DEV))
    other, same = SK.lm_head_greedy(*args, **kw, rules=rules)
    assert torch.equal(bits(logits), bits(same))
    logits = logits.float().reshape(-1)
    logits[int(tok)] = -torch.inf
    assert int(other) == int(logits.argmax())
