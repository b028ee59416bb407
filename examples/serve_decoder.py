"""A decoder of tensor-ring projections served over a paged cache.

    python examples/serve_decoder.py [--layers 2] [--tokens 32] [--graph]

Random weights; the point is the order of the calls in a serving step:

    plan_step -> per layer: q, k, v projections -> append_kv -> paged_attention -> o projection
    -> residual_norm -> gated MLP -> residual_norm -> logits -> sample_tokens

Prompts of different lengths are prefilled in one step; then every request decodes, one token a
step.  Nothing in a step waits for the GPU: with --graph the decode step is captured once in a
CUDA graph and replayed.
"""
from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from kernel_task_b200 import (TRSpec, append_kv, paged_attention, plan_step,  # noqa: E402
                              prepare_optimized, release_pages, residual_norm, sample_tokens)
from kernel_task_b200.spec import baseline_cores  # noqa: E402


@dataclass(frozen=True)
class Shape:
    """Modes of the projections (each a product of three) and the heads they make."""

    hidden: tuple[int, int, int] = (4, 8, 16)
    inner: tuple[int, int, int] = (8, 8, 16)
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    rank: int = 8
    vocab: int = 2053
    layers: int = 2
    page_size: int = 16

    def specs(self) -> dict[str, TRSpec]:
        q = (self.heads, 8, self.head_dim // 8)
        kv = (self.kv_heads, 8, self.head_dim // 8)
        return {"q": TRSpec(self.hidden, q, self.rank), "k": TRSpec(self.hidden, kv, self.rank),
                "v": TRSpec(self.hidden, kv, self.rank), "o": TRSpec(q, self.hidden, self.rank),
                "gate": TRSpec(self.hidden, self.inner, self.rank),
                "up": TRSpec(self.hidden, self.inner, self.rank),
                "down": TRSpec(self.inner, self.hidden, self.rank)}


class Decoder:
    """Weights, the paged cache and its bookkeeping for up to `requests` requests."""

    def __init__(self, shape: Shape, requests: int, pages: int, longest: int, *, seed: int = 0,
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda"):
        self.shape, self.dtype = shape, dtype
        specs = shape.specs()
        width = specs["q"].in_features
        self.cores = [{n: baseline_cores(s, seed=100 * layer + i, dtype=dtype, device=device)
                       for i, (n, s) in enumerate(specs.items())} for layer in range(shape.layers)]
        self.ops = [{n: prepare_optimized(c[n], specs[n]) for n in specs} for c in self.cores]
        g = torch.Generator().manual_seed(seed)

        def normal(*size, scale=1.0, shift=0.0):
            return (torch.randn(*size, generator=g) * scale + shift).to(device, dtype)

        self.embed = normal(shape.vocab, width)
        self.head = normal(shape.vocab, width, scale=3 * width ** -0.5)
        # norms before and after attention and MLP; a gate of attention and one of the MLP
        self.norms = [{n: normal(width, scale=0.05, shift=1.0)
                       for n in ("attn_pre", "attn_post", "mlp_pre", "mlp_post")}
                      for _ in range(shape.layers)]
        self.gates = [{n: normal(width, scale=0.1, shift=0.5) for n in ("attn", "mlp")}
                      for _ in range(shape.layers)]
        self.final = normal(width, scale=0.05, shift=1.0)

        pool = (shape.layers, pages, shape.kv_heads, shape.page_size, shape.head_dim)
        self.k_pages = torch.empty(pool, dtype=dtype, device=device)
        self.v_pages = torch.empty(pool, dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.tables = torch.full((requests, -(-longest // shape.page_size)), -1, **ints)
        self.lens = torch.zeros(requests, **ints)
        self.free = torch.arange(pages - 1, -1, -1, **ints)
        self.free_count = torch.tensor([pages], **ints)

    def forward(self, ids: torch.Tensor, new: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Logits of each request's last token in the step, and which requests got their pages.

        ids: the step's tokens, request by request; new [requests]: how many each brings."""
        s = self.shape
        step = plan_step(self.lens, new, self.tables, self.free, self.free_count, s.page_size,
                         ids.numel(), inplace=True)
        h = self.embed[ids]
        _, x = residual_norm(None, h, pre=self.norms[0]["attn_pre"])
        for layer, (op, norm, gate) in enumerate(zip(self.ops, self.norms, self.gates)):
            heads = (-1, s.head_dim)
            append_kv(op["k"](x).unflatten(1, heads), op["v"](x).unflatten(1, heads),
                      self.k_pages[layer], self.v_pages[layer], step.slots)
            seen = paged_attention(op["q"](x).unflatten(1, heads), self.k_pages[layer],
                                   self.v_pages[layer], self.tables, step.lens, step.starts)
            h, x = residual_norm(op["o"].accumulate(seen.flatten(1)), h, post=norm["attn_post"],
                                 gate=gate["attn"], pre=norm["mlp_pre"])
            inner = op["up"].forward_silu_mul(x, op["gate"].accumulate(x))
            last = layer + 1 == s.layers
            h, x = residual_norm(op["down"].accumulate(inner), h, post=norm["mlp_post"],
                                 gate=gate["mlp"],
                                 pre=self.final if last else self.norms[layer + 1]["attn_pre"])
        return x[(step.starts[1:] - 1).clamp(min=0)] @ self.head.t(), step.granted

    def step(self, ids: torch.Tensor, new: torch.Tensor, noise: torch.Tensor,
             temperature: torch.Tensor, **limits) -> torch.Tensor:
        """The next token of every request; -1 where it brings none or did not get its pages."""
        logits, granted = self.forward(ids, new)
        drawn = sample_tokens(logits, noise, temperature, **limits)[0]
        return torch.where((granted > 0) & (new > 0), drawn, -1)

    def finish(self, done: torch.Tensor) -> None:
        """Give back the pages of the requests with done[r] != 0."""
        release_pages(self.lens, done, self.tables, self.free, self.free_count,
                      self.shape.page_size)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=32, help="tokens to decode after the prompts")
    ap.add_argument("--graph", action="store_true", help="replay the decode step from a CUDA graph")
    a = ap.parse_args()
    shape = Shape(layers=a.layers)
    prompts = [5, 130, 33, 260]
    R = len(prompts)
    model = Decoder(shape, R, pages=256, longest=1024)
    g = torch.Generator(device="cuda").manual_seed(1)
    ints = dict(dtype=torch.int32, device="cuda")
    noise = torch.empty(R, shape.vocab, device="cuda")
    heat = torch.full((R,), 0.8, device="cuda")
    limits = dict(top_k=torch.full((R,), 50, **ints), top_p=torch.full((R,), 0.95, device="cuda"))

    ids = torch.randint(shape.vocab, (sum(prompts),), generator=g, device="cuda")
    noise.exponential_(generator=g)
    ids = model.step(ids, torch.tensor(prompts, **ints), noise, heat, **limits)
    out = [ids.clone()]
    one = torch.ones(R, **ints)
    ids = ids.clone()
    replay = None
    if a.graph:
        kept = [t.clone() for t in (model.lens, model.tables, model.free_count)]
        model.step(ids, one, noise, heat, **limits)  # warm up, then take the bookkeeping back
        for t, k in zip((model.lens, model.tables, model.free_count), kept):
            t.copy_(k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ids.copy_(model.step(ids, one, noise, heat, **limits))
        replay = graph.replay
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.tokens):
        noise.exponential_(generator=g)
        if replay:
            replay()
        else:
            ids = model.step(ids, one, noise, heat, **limits)
        out.append(ids.clone())
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / max(a.tokens, 1) * 1e6
    print(f"{R} requests, {a.layers} layers: {took:.0f} us a decode step; lengths "
          f"{model.lens.tolist()}, free pages {int(model.free_count)}")
    for r, row in enumerate(torch.stack(out, 1).tolist()):
        print(f"request {r}: {row[:12]} ...")
    model.finish(one)
    print(f"finished: free pages {int(model.free_count)}")


if __name__ == "__main__":
    main()
