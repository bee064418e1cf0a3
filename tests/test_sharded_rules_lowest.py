"""The row-sharded head's choice where every allowed logit is minus infinity:
an allowed token all the same, the first of them, though ranks before it allow
none and say minus infinity too (gloo ranks on the CPU, and one rank on a GPU
with the kernels, tests/test_sharded_rules_gpu.py)."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from oracle import logits as R
from spectra_b200.sharded import ShardedW4A16Linear
from tests.test_sharded import _free_port, _layer, _oracle_local
from tests.test_sharded_rules import argmax_under

N, K = 203, 64
# The allowed tokens of each row (biased to minus infinity) and the choice: of 4 ranks 0-50, 51-101, 102-152, 153-202.
ROWS = [([N - 2], N - 2), ([60], 60), ([110, 120, 201], 110), ([3], 3), ([], -1), ([52, 190], 52)]


def rules():
    out = []
    for tokens, _ in ROWS:
        allowed = np.zeros(N, bool)
        allowed[tokens] = True
        out.append(dict(biases=[(t, -np.inf) for t in tokens], allowed=allowed))
    return out


def run():
    p, s, z, idx, ow, bias = _layer(N, K, 3, 11)
    lin = ShardedW4A16Linear(p, s, z, outlier_idx=idx, outlier_w=ow, bias=bias, marlin_layout=True, device=torch.device("cpu"),
                             local_fn=_oracle_local, argmax_fn=argmax_under)
    return lin.greedy(torch.randn(len(ROWS), K, generator=torch.Generator().manual_seed(11)).to(torch.float16), rules=rules()).tolist()


def worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        q.put((rank, run()))
    finally:
        dist.destroy_process_group()


def test_the_oracle_chooses_the_first_allowed():
    for r, (_, want) in zip(rules(), ROWS):
        assert R.adjust(np.zeros(N, np.float32), **r)[1] == want


@pytest.mark.parametrize("world", [1, 2, 4])
def test_an_allowed_token_of_minus_infinity(world):
    expect = [w for _, w in ROWS]
    if world == 1:
        assert run() == expect
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
