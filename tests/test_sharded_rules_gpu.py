"""ShardedW4A16Linear.greedy(rules=) with the kernels: one rank, and two ranks'
slices put together as the exchange does, against the rules' oracle on the
head's own logits."""
import numpy as np
import pytest
import torch

from oracle import logits as R
from spectra_b200 import kernels as SK
from spectra_b200.logits import LogitRules
from spectra_b200.sharded import ShardedW4A16Linear, shard_bounds

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")
N, K = 4099, 2048


def head(seed):
    from tests.helpers import random_format
    f = random_format(N, K, 21, seed=seed, ow_dtype="bf16")
    return ShardedW4A16Linear(torch.from_numpy(f["packed"]), torch.from_numpy(f["scales"]), torch.from_numpy(f["zeros"]),
                              outlier_idx=torch.from_numpy(f["outlier_idx"]), outlier_w=f["outlier_w_t"], marlin_layout=True, device=DEV)


def rules_of(M, seed):
    """Per row as the oracle takes them, and the device's."""
    rng = np.random.default_rng(seed)
    rows = []
    for m in range(M):
        allowed = rng.random(N) < (1.0, 0.5, 0.002, 0.0)[m % 4]
        biases = [(int(rng.integers(0, N)), float(np.float32(rng.normal() * 3))) for _ in range(5)]
        if m % 4 == 2:  # one allowed token, at minus infinity
            allowed[:] = False
            allowed[N - 2] = True
            biases[4] = (N - 2, -np.inf)
        rows.append(dict(ids=rng.integers(0, N, 60).tolist(), prompt=20, repetition=1.25, frequency=0.125, presence=0.25,
                         biases=biases, allowed=allowed))
    i32 = lambda x: torch.tensor(np.array(x), dtype=torch.int32, device=DEV)  # noqa: E731
    bits = np.zeros((M, -(-N // 32) * 32), bool)
    bits[:, :N] = [r["allowed"] for r in rows]
    words = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    dev = LogitRules(ids=i32([r["ids"] for r in rows]), prompt_lengths=i32([20] * M), repetition=1.25, frequency=0.125,
                     presence=0.25, bias_ids=i32([[t for t, _ in r["biases"]] for r in rows]),
                     bias=torch.tensor([[v for _, v in r["biases"]] for r in rows], dtype=torch.float32, device=DEV),
                     allowed=torch.from_numpy(words.copy()).to(DEV))
    return rows, dev


@pytest.mark.parametrize("M", [1, 8, 33])
def test_one_rank_and_captured(M):
    lin = head(3)
    rows, rules = rules_of(M, M)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(DEV)
    got = lin.greedy(x, rules=rules)
    logits = lin.forward(x)
    want = [R.adjust(y, **r)[1] for y, r in zip(logits.float().cpu().numpy(), rows)]
    assert got.tolist() == want and (M < 4 or (want[2] == N - 2 and want[3] == -1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = lin.greedy(x, rules=rules)
    for seed in (50, 51):
        x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        assert torch.equal(tokens, lin.greedy(x, rules=rules))


@pytest.mark.parametrize("world", [2, 5])
def test_slices_of_the_vocabulary_give_the_whole_rows_choice(world):
    M = 8
    lin = head(4)
    rows, rules = rules_of(M, 9)
    logits = lin.forward(torch.randn(M, K, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(DEV))
    want = [R.adjust(y, **r)[1] for y, r in zip(logits.float().cpu().numpy(), rows)]
    pairs = []
    for rank in range(world):
        _, lo, hi = shard_bounds(N, world, rank)
        pairs.append(SK.argmax(logits[:, lo:hi], idx_offset=lo, with_values=True, rules=rules))
    for m in range(M):
        allowed = [(float(v[m]), int(i[m])) for i, v in pairs if int(i[m]) >= 0]
        best = max((v for v, _ in allowed), default=None)
        assert next((i for v, i in allowed if v == best), -1) == want[m]
        for (i, v), (_, lo, hi) in zip(pairs, (shard_bounds(N, world, r) for r in range(world))):
            if int(i[m]) < 0:  # none of the slice's tokens is allowed
                assert float(v[m]) == -np.inf and not rows[m]["allowed"][lo:hi].any()
