"""Workspaces of captured calls: a graph zeroes what it relies on by itself, in
whatever order graphs are replayed, and eager calls never use a graph's."""
import pytest
import torch

from spectra_b200 import _lib as L
from spectra_b200 import kernels as SK
from spectra_b200 import paged as PG
from tests.helpers import act, random_format
from tests.test_paged_gpu import DEV, Step, draw

pytestmark = pytest.mark.gpu


class DirtyPool:
    """A fresh capture stream and a graph memory pool whose free memory holds 0xFF."""

    def __init__(self, nbytes=96 << 20):
        self.stream, self.pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
        self.first = self.capture(lambda: torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV).view(-1)[:0])[0]
        self.first.replay()
        torch.cuda.synchronize()

    def capture(self, call):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=self.pool, stream=self.stream):
            out = call()
        return graph, out


def split_step():
    st = Step([9011, 3, 7000], [1] * 3, 8, 2, 128, 64, "bf16", seed=31)
    st.fill()
    return st, draw((3, 8, 128), 32, "bf16").to(DEV)


def test_capture_id():
    s = torch.cuda.Stream()
    ident = L.lib().spectra_stream_capture_id
    assert ident(s.cuda_stream) == 0 and ident(None) == 0
    ids = []
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            ids.append(ident(s.cuda_stream))
            assert ident(torch.cuda.default_stream().cuda_stream) == 0
            torch.zeros(1, device=DEV)
    assert ids[0] and ids[1] and ids[0] != ids[1] and ident(s.cuda_stream) == 0


def test_paged_attention_captured_on_a_stream_without_a_workspace():
    st, q = split_step()
    want = PG.paged_attention(q, st.cache, st.batch)
    assert want.any()
    p = DirtyPool()
    a, out_a = p.capture(lambda: PG.paged_attention(q, st.cache, st.batch))
    b, out_b = p.capture(lambda: (PG.paged_attention(q, st.cache, st.batch), PG.paged_attention(q, st.cache, st.batch)))
    with torch.cuda.stream(p.stream):  # an eager call of that stream, before any replay
        eager = PG.paged_attention(q, st.cache, st.batch)
    torch.cuda.synchronize()
    assert torch.equal(eager, want)
    for graph, outs in ((b, out_b), (a, (out_a,)), (b, out_b), (b, out_b)):  # the later one first
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        del outs


def test_graphs_of_paged_attention_with_their_own_workspaces_may_overlap():
    st, q = split_step()
    want = PG.paged_attention(q, st.cache, st.batch)
    stream = torch.cuda.Stream()
    graphs = []
    for _ in range(2):  # (own pools; each many calls long, so that replays do overlap)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = [PG.paged_attention(q, st.cache, st.batch) for _ in range(40)]
        graphs.append((graph, outs))
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (graph, outs), side in zip(graphs, sides):
            with torch.cuda.stream(side):
                for o in outs:
                    o.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(o, want) for o in outs)


def test_split_gemm_captured_on_a_stream_without_a_large_enough_workspace():
    def problem(M, N, K, seed):
        fmt = random_format(N, K, 0, seed=seed, ow_dtype="bf16")
        w = [torch.from_numpy(fmt[n]).to(DEV) for n in ("packed", "scales", "zeros")]
        a = act(M, K, seed=seed + 1, dtype="bf16").to(DEV)
        assert L.lib().spectra_w4a16_gemm_workspace_bytes(M, N, K, 0) > 0
        return lambda: SK.batched_w4a16_gemm(a, *w, marlin_layout=True)

    small, large = problem(16, 256, 16384, 41), problem(256, 1024, 4096, 43)  # (over 1 MB of partials)
    want = [small(), large()]
    p = DirtyPool()
    a, out_a = p.capture(lambda: [small()])
    b, out_b = p.capture(lambda: [small(), large()])
    with torch.cuda.stream(p.stream):
        eager = small()  # before any replay
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0])
    c, out_c = p.capture(lambda: [large(), small()])  # the stream's own is too small for the first
    torch.cuda.synchronize()
    for graph, outs, wants in ((c, out_c, want[::-1]), (b, out_b, want), (a, out_a, want[:1]), (b, out_b, want)):
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
