"""Greedy generation for several sequences at once on the paged INT4 KV cache.

A Llama-shaped model of random weights: W4A16 linears and embedding
(spectra_b200.modules), and per layer rotate-and-append and attention on a
paged cache (spectra_b200.paged).  Prompts of different lengths go through in
one ragged batch, then every step appends one token per sequence; the step is
captured in a CUDA graph and replayed.

    python examples/paged_generate.py --layers 2 --hidden 512 --tokens 32
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import List

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from spectra_b200 import compress as C  # noqa: E402
from spectra_b200 import kernels as SK  # noqa: E402
from spectra_b200 import paged  # noqa: E402
from spectra_b200.modules import SpectraFusedEmbedding, SpectraFusedLinear  # noqa: E402


def _linear(n: int, k: int, gen: torch.Generator, std: float) -> SpectraFusedLinear:
    c = C.compress_linear((torch.randn(n, k, generator=gen, device="cuda") * std).to(torch.float16))
    m = SpectraFusedLinear(k, n, marlin_layout=True)
    m.set_weights(c.packed, c.scales, c.zeros, outlier_idx=c.outlier_idx, outlier_weight=c.outlier_w, marlin_layout=True)
    return m


class PagedLlama:
    """Random-weight decoder whose attention lives on paged INT4 caches, one per layer."""

    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, inner=1536, vocab=1024, pages=64,
                 page_size=64, max_len=1024, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.page_size, self.max_len = heads, kv_heads, head_dim, page_size, max_len
        std = hidden ** -0.5
        q, kv = heads * head_dim, kv_heads * head_dim
        shapes = dict(q=(q, hidden), k=(kv, hidden), v=(kv, hidden), o=(hidden, q), gate=(inner, hidden),
                      up=(inner, hidden), down=(hidden, inner))
        self.layers = [{n: _linear(*s, g, s[1] ** -0.5) for n, s in shapes.items()} for _ in range(layers)]
        c = C.compress_linear((torch.randn(vocab, hidden, generator=g, device="cuda") * std).to(torch.float16))
        self.embed = SpectraFusedEmbedding(vocab, hidden, marlin_layout=True)
        self.embed.set_weights(c.packed, c.scales, c.zeros, c.outlier_idx, c.outlier_w, marlin_layout=True)
        self.embed.target_dtype = torch.bfloat16
        self.head = SpectraFusedLinear(hidden, vocab, marlin_layout=True)
        self.head.set_weights(c.packed, c.scales, c.zeros, outlier_idx=c.outlier_idx, outlier_weight=c.outlier_w,
                              marlin_layout=True)
        self.caches = [paged.PagedKVCache(pages, kv_heads, head_dim, page_size) for _ in range(layers)]
        self.free = list(range(pages))
        freq = 500000.0 ** (-torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float64) / head_dim)
        angle = torch.arange(max_len, device="cuda", dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    @staticmethod
    def _norm(x: torch.Tensor) -> torch.Tensor:
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)

    def forward(self, ids: torch.Tensor, batch: paged.TokenBatch) -> torch.Tensor:
        """Hidden states [T, hidden] of the batch's new tokens; their keys and values enter the caches."""
        x = self.embed(ids)
        for w, cache in zip(self.layers, self.caches):
            h = self._norm(x)
            q, k, v = (w[n](h).unflatten(-1, (-1, self.head_dim)) for n in "qkv")
            q = paged.paged_kv_append(cache, batch, k, v, q=q, cos=self.cos, sin=self.sin)
            x = x + w["o"](paged.paged_attention(q, cache, batch).flatten(1))
            h = self._norm(x)
            x = x + w["down"](torch.nn.functional.silu(w["gate"](h)) * w["up"](h))
        return self._norm(x)

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return self.head(hidden)

    def tables(self, lens: List[int]) -> torch.Tensor:
        """Pages for sequences of these lengths, taken from the free ones."""
        need = [-(-n // self.page_size) for n in lens]
        if sum(need) > len(self.free):
            raise RuntimeError(f"{sum(need)} pages wanted, {len(self.free)} free")
        rows = [[self.free.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need]
        return torch.tensor(rows, dtype=torch.int32, device="cuda")

    def release(self, tables: torch.Tensor) -> None:
        self.free += [p for p in tables.flatten().tolist() if p >= 0]

    @torch.no_grad()
    def generate(self, prompts: List[List[int]], tokens: int, graph: bool = True):
        """Greedy continuations [B, tokens], and the logits each was chosen from [B, tokens, vocab]."""
        lens = [len(p) for p in prompts]
        if not lens or min(lens) < 1 or tokens < 1:
            raise ValueError("prompts of one token at least, and one token to generate")
        # positions from max_len on have no angles and are not kept (the last token generated is not appended)
        if max(lens) + tokens - 1 > self.max_len:
            raise ValueError(f"a prompt of {max(lens)} and {tokens} tokens pass max_len={self.max_len}")
        tables = self.tables([n + tokens for n in lens])
        try:
            return self._generate(prompts, lens, tables, tokens, graph)
        finally:
            self.release(tables)

    def _generate(self, prompts, lens, tables, tokens, graph):
        seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
        ids = torch.tensor([t for p in prompts for t in p], device="cuda")
        prompt = paged.TokenBatch(tables, seq_lens, cu_q=cu, total=sum(lens), max_q=max(lens), max_len=self.max_len)
        hidden = self.forward(ids, prompt)
        logits = self.logits(hidden[cu[1:].long() - 1])
        step = paged.TokenBatch(tables, seq_lens, max_len=self.max_len)  # one token per sequence from here on
        last = SK.argmax(logits)

        def decode() -> None:
            seq_lens.add_(1)
            logits.copy_(self.logits(self.forward(last, step)))
            last.copy_(SK.argmax(logits))

        out, chosen_from = [last.clone()], [logits.clone()]
        replay = decode
        for i in range(1, tokens):
            if graph and i == 2:  # (one eager step first: workspaces and kernel attributes)
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                keep = seq_lens.clone(), last.clone()
                with torch.cuda.stream(side):
                    decode()  # this stream's workspaces; the token is written again below
                torch.cuda.current_stream().wait_stream(side)
                seq_lens.copy_(keep[0])
                last.copy_(keep[1])
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    decode()
                replay = captured.replay
            replay()
            out.append(last.clone())
            chosen_from.append(logits.clone())
        return torch.stack(out, 1), torch.stack(chosen_from, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--prompts", type=int, nargs="+", default=[17, 200, 64, 1], help="prompt lengths")
    a = ap.parse_args()
    model = PagedLlama(layers=a.layers, hidden=a.hidden)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in a.prompts]
    tokens, _ = model.generate(prompts, a.tokens)
    for n, row in zip(a.prompts, tokens.tolist()):
        print(f"after {n} tokens: {row}")


if __name__ == "__main__":
    main()
