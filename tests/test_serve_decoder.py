"""GPU: the example decoder (examples/serve_decoder.py), the serving operators and the tensor-ring
projections run together, against a numpy float64 decoder of the same weights without a cache.

Tolerance.  Two layers round some fourteen intermediate tensors to bf16 (unit 2^-8, rms 0.29 of a
unit each way) along the path of every value: 14 ** 0.5 * 2^-8 * 0.58 = 0.9 % of the logits'
norm if nothing amplified; the bound is 4 %."""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import oracle
from oracle import serve_oracle as so

pytestmark = pytest.mark.gpu


def load_example():
    path = Path(__file__).resolve().parents[1] / "examples" / "serve_decoder.py"
    spec = importlib.util.spec_from_file_location("serve_decoder", path)
    module = importlib.util.module_from_spec(spec)
    sys.modules["serve_decoder"] = module
    spec.loader.exec_module(module)
    return module


def f64(t):
    return t.double().cpu().numpy()


def reference_logits(model, ids):
    """Logits of every position of one sequence."""
    s = model.shape

    def tr(layer, name, x):
        return oracle.tr_forward_reference(x, [f64(c) for c in model.cores[layer][name]])

    h = f64(model.embed)[ids]
    x = so.residual_norm(None, h, pre=f64(model.norms[0]["attn_pre"]))[1]
    n = len(ids)
    for layer in range(s.layers):
        norm = {k: f64(v) for k, v in model.norms[layer].items()}
        gate = {k: f64(v) for k, v in model.gates[layer].items()}
        q = tr(layer, "q", x).reshape(n, s.heads, s.head_dim)
        k = tr(layer, "k", x).reshape(n, s.kv_heads, s.head_dim)
        v = tr(layer, "v", x).reshape(n, s.kv_heads, s.head_dim)
        out = np.zeros_like(q)
        for i in range(n):
            for head in range(s.heads):
                kv = head // (s.heads // s.kv_heads)
                a = k[:i + 1, kv] @ q[i, head] / math.sqrt(s.head_dim)
                e = np.exp(a - a.max())
                out[i, head] = e @ v[:i + 1, kv] / e.sum()
        h, x = so.residual_norm(tr(layer, "o", out.reshape(n, -1)), h, post=norm["attn_post"],
                                gate=gate["attn"], pre=norm["mlp_pre"])
        g = tr(layer, "gate", x)
        inner = g / (1 + np.exp(-g)) * tr(layer, "up", x)
        nxt = f64(model.final) if layer + 1 == s.layers else f64(model.norms[layer + 1]["attn_pre"])
        h, x = so.residual_norm(tr(layer, "down", inner), h, post=norm["mlp_post"], gate=gate["mlp"],
                                pre=nxt)
    return x @ f64(model.head).T


def test_decoder_against_a_decoder_without_a_cache():
    ex = load_example()
    model = ex.Decoder(ex.Shape(), 3, pages=24, longest=160)
    rng = np.random.default_rng(0)
    lengths, grown = [5, 71, 33], 4
    seqs = [rng.integers(0, model.shape.vocab, n + grown) for n in lengths]
    want = [reference_logits(model, s) for s in seqs]

    def close(got, rows):
        for r, at in enumerate(rows):
            err = np.linalg.norm(f64(got[r]) - want[r][at]) / np.linalg.norm(want[r][at])
            assert err <= 0.04, (r, at, err)

    ints = dict(dtype=torch.int32, device="cuda")
    prompt = torch.tensor(np.concatenate([s[:n] for s, n in zip(seqs, lengths)]), device="cuda")
    got, granted = model.forward(prompt, torch.tensor(lengths, **ints))
    assert granted.tolist() == [1, 1, 1]
    close(got, [n - 1 for n in lengths])
    for i in range(grown - 2):  # a token each
        ids = torch.tensor([s[n + i] for s, n in zip(seqs, lengths)], device="cuda")
        got, _ = model.forward(ids, torch.ones(3, **ints))
        close(got, [n + i for n in lengths])
    # two tokens for the second request, none for the first, one for the third
    ids = torch.tensor([seqs[1][lengths[1] + 2], seqs[1][lengths[1] + 3], seqs[2][lengths[2] + 2]],
                       device="cuda")
    got, _ = model.forward(ids, torch.tensor([0, 2, 1], **ints))
    err = [np.linalg.norm(f64(got[r]) - want[r][at]) / np.linalg.norm(want[r][at])
           for r, at in ((1, lengths[1] + 3), (2, lengths[2] + 2))]
    assert max(err) <= 0.04, err
    assert model.lens.tolist() == [7, 75, 36]
    model.finish(torch.tensor([1, 1, 1], **ints))
    assert int(model.free_count) == 24 and model.lens.tolist() == [0, 0, 0]
    assert sorted(model.free.tolist()) == list(range(24))


def test_decode_step_from_a_graph_gives_the_same_tokens():
    ex = load_example()
    ints = dict(dtype=torch.int32, device="cuda")
    one = torch.ones(2, **ints)
    heat, k = torch.full((2,), 0.9, device="cuda"), torch.full((2,), 40, **ints)
    g = torch.Generator(device="cuda").manual_seed(3)
    noises = [torch.empty(2, ex.Shape().vocab, device="cuda").exponential_(generator=g)
              for _ in range(7)]
    prompt = torch.arange(50, device="cuda")

    def begin():
        model = ex.Decoder(ex.Shape(), 2, pages=16, longest=96)
        return model, model.step(prompt, torch.tensor([20, 30], **ints), noises[0], heat, top_k=k)

    model, ids = begin()
    want = []
    for n in noises[1:]:
        ids = model.step(ids, one, n, heat, top_k=k)
        want.append(ids.tolist())
    model, ids = begin()
    ids, noise = ids.clone(), noises[1].clone()
    kept = [t.clone() for t in (model.lens, model.tables, model.free_count)]
    model.step(ids, one, noise, heat, top_k=k)
    for t, v in zip((model.lens, model.tables, model.free_count), kept):
        t.copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids.copy_(model.step(ids, one, noise, heat, top_k=k))
    got = []
    for n in noises[1:]:
        noise.copy_(n)
        graph.replay()
        got.append(ids.tolist())
    assert got == want
    assert model.lens.tolist() == [26, 36]
