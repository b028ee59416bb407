"""The serving operators where a wrong answer, a needless refusal or an unsafe access would hide:
the sizes at which launches change shape, extreme parameters, and state that outlives a call.

Tolerances are those of test_serve.py."""
from __future__ import annotations

import pytest
import torch

import kernel_task_b200 as trb
from test_serve import check_sample, i32, sample_inputs

gpu = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------- sampling
@gpu
@pytest.mark.parametrize("vocab", [2049, 4097, 8193, 16391])
def test_sample_rows_split_over_a_cluster_on_a_busy_gpu(vocab):
    """A row is cut over 2, 4 or 8 blocks, which store into one another's shared memory; while
    other work holds SMs the blocks of a cluster may start apart."""
    logits, noise = sample_inputs(3, vocab, torch.float32, vocab)
    heat, k = torch.ones(3, device=DEV), i32([0, 40, 900])
    p = torch.tensor([0.9, 1.0, 0.8], device=DEV)
    want = check_sample(logits, noise, heat, top_k=k, top_p=p)
    busy, x = torch.cuda.Stream(), torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        with torch.cuda.stream(busy):
            x.mul_(1.0)
        got.append(trb.sample_tokens(logits, noise, heat, top_k=k, top_p=p)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
