"""The row-sharded head's greedy choice under rules on the logits, on 2 and 4
gloo ranks (CPU): every rank applies the rules to its slice of the vocabulary
(here by the oracle), and the pairs give the choice of the whole row."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from oracle import logits as R
from spectra_b200.sharded import ShardedW4A16Linear
from tests.test_sharded import _free_port, _layer, _oracle_local

N, K, M = 203, 64, 5


def rules_of(seed):
    """Per row: ids, their prompt's length, biases, allowed."""
    rng = np.random.default_rng(seed)
    rows = []
    for m in range(M):
        ids = rng.integers(0, N, 60).tolist()
        allowed = rng.random(N) < (1.0, 0.5, 0.03, 0.0, 0.01)[m]
        if m == 4:
            allowed[:] = False
            allowed[N - 2] = True  # one token, of the last rank that has any
        rows.append(dict(ids=ids, prompt=20, repetition=1.4, frequency=0.1, presence=0.2,
                         biases=[(int(rng.integers(0, N)), float(rng.normal() * 3)) for _ in range(5)], allowed=allowed))
    return rows


def argmax_under(y, offset, rules=None):
    val, idx = [], []
    for row, r in zip(y.float().numpy(), rules):
        x, token = R.adjust(row, offset=offset, **r)
        idx.append(token)
        val.append(x[token - offset] if token >= 0 else -np.inf)
    return torch.tensor(val, dtype=torch.float32), torch.tensor(idx, dtype=torch.int64)


def worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        q.put((rank, run(7)))
    finally:
        dist.destroy_process_group()


def run(seed):
    p, s, z, idx, ow, bias = _layer(N, K, 3, seed)
    lin = ShardedW4A16Linear(p, s, z, outlier_idx=idx, outlier_w=ow, bias=bias, marlin_layout=True, device=torch.device("cpu"),
                             local_fn=_oracle_local, argmax_fn=argmax_under)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(torch.float16)
    x[4] = float("-inf")  # logits of minus infinity or NaN: an allowed token is chosen all the same
    return lin.greedy(x, rules=rules_of(seed)).tolist()


def want(seed):
    p, s, z, idx, ow, bias = _layer(N, K, 3, seed)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(torch.float16)
    x[4] = float("-inf")
    full = _oracle_local(x, p, s, z, idx, ow, bias, True).float().numpy()
    return [R.adjust(row, **r)[1] for row, r in zip(full, rules_of(seed))]


@pytest.mark.parametrize("world", [1, 2, 4])
def test_the_choice_of_the_whole_row(world):
    expect = want(7)
    assert expect[3] == -1 and expect[4] == N - 2
    if world == 1:
        assert run(7) == expect
        return
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
    assert all(got[r] == expect for r in range(world))
