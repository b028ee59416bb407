"""The serving operators where a wrong answer, a needless refusal or an unsafe access would hide:
the sizes at which launches change shape, extreme parameters, and state that outlives a call.

Tolerances are those of test_serve.py."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import kernel_task_b200 as trb
from kernel_task_b200 import abi
from test_serve import (attention_case, check_attention, check_plan, check_sample, f64, gen, i32,
                        make_pool, sample_inputs)
from test_serve_decoder import load_example
from test_serve_limits import attention_struct, need_of

gpu = pytest.mark.gpu
DEV = "cuda"
TESTS = Path(__file__).resolve().parent


def in_fresh_process(call, **env):
    """Runs `call` of this file where no earlier call has raised a limit or kept a workspace."""
    code = f"import sys; sys.path[:0] = [{str(TESTS)!r}, {str(TESTS.parent)!r}]\n" \
           f"import test_serve_edges as t\nt.{call}"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, **env})
    assert r.returncode == 0, r.stdout + r.stderr


# ------------------------------------------------------------------------------ step plan
def plans_of(sizes):
    for requests in sizes:
        check_plan([1] * requests, [1] * requests, 16, 2, requests)
        check_plan([16] * requests, [1] * requests, 16, 2, requests)


def releases_of(sizes):
    for requests in sizes:
        lens = [17] * requests
        tables, free, total = make_pool(lens, 16, 2, 3)
        pool = np.full(total, -1, np.int32)
        pool[:3] = free
        d = dict(lens=i32(lens), tables=i32(tables), free=i32(pool), count=i32([3]))
        trb.release_pages(d["lens"], i32([1] * requests), d["tables"], d["free"], d["count"], 16)
        assert d["free"].cpu().tolist() == list(free) + tables.flatten().tolist()
        assert int(d["count"]) == total and not d["lens"].any()


@gpu
@pytest.mark.parametrize("call", ["plans_of([4074, 4073, 4095, 4096, 16384, 4095])",
                                  "plans_of([4095])",
                                  "releases_of([12225, 12224, 12288, 12289, 16384, 12288])",
                                  "releases_of([12288])"])
def test_requests_where_shared_memory_passes_the_default(call):
    in_fresh_process(call)


# ------------------------------------------------------------------------------ attention
@gpu
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("dtype,dim", [(torch.float32, 40), (torch.bfloat16, 40),
                                       (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_scores_that_pass_fp32_downwards(new, dtype, dim):
    """The first keys' scores are -inf in fp32: their probability is 0, as in 64 bits."""
    q, kp, vp, tables, lens, starts = attention_case([100], [new], 4, 2, dim, 16, dtype)
    kp[int(tables[0, 0]), :, :3, 0] = -3e38
    kp[int(tables[0, 5]), :, 2, 0] = -3e38
    check_attention((q.abs() + 1, kp, vp, tables, lens, starts))


@gpu
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("dim", [40, 64, 128])
def test_attention_log_sum_of_a_nan_row_is_nan(new, dim):
    """-inf would say that the row saw nothing, and a join by log-sums would drop the NaN."""
    args = attention_case([100], [new], 4, 2, dim, 16, torch.bfloat16)
    want, want_lse = trb.paged_attention(*args, return_lse=True)
    q = args[0].clone()
    q[0, 1] = math.nan
    out, lse = trb.paged_attention(q, *args[1:], return_lse=True)
    assert out[0, 1].isnan().all() and lse[0, 1].isnan()
    out[0, 1], lse[0, 1] = want[0, 1], want_lse[0, 1]
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def long_chunks():
    """Prompts and chunks over all SMs, some items shared by blocks; the inputs pass L2 out."""
    args = attention_case([3000, 2500, 260], [600, 500, 260], 16, 4, 128, 16, torch.bfloat16)
    torch.cuda.synchronize()
    torch.empty(64 << 20, device=DEV).fill_(1.0)
    return args


def assert_right_or_nan(out, lse, want, want_lse):
    """By element: a block that spoils an item it had done its part of may do so while the block
    that joins the parts writes them, all of them right."""
    for got, right in ((out, want), (lse, want_lse)):
        assert (got.isnan() | (got == right)).all()
    return int(out.isnan().sum())


@gpu
def test_attention_timeout_spoils_what_it_leaves_until_the_state_is_zeroed():
    args = long_chunks()
    few = attention_case([3000, 40], [1, 1], 16, 4, 128, 16, torch.bfloat16)
    want, want_lse = trb.paged_attention(*args, return_lse=True)
    few_want = trb.paged_attention(*few)
    out, lse = torch.full_like(want, 7.0), torch.full_like(want_lse, 7.0)
    few_out = torch.full_like(few_want, 7.0)
    a, b = attention_struct(args, out, lse, wait_polls=1), attention_struct(few, few_out)
    need, stream = max(need_of(a), need_of(b)), torch.cuda.current_stream().cuda_stream
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)

    def call(s):
        abi.check(abi.lib().tr_paged_attention(ctypes.byref(s), ctypes.c_void_p(ws.data_ptr()), need,
                                               ctypes.c_void_p(stream)), "tr_paged_attention")

    def status():
        return abi.workspace_status(ws.data_ptr(), need, reset=False, stream=stream)

    for polls in (32, 8, 4, 3, 2):  # ends anywhere, or not at all
        a.wait_polls = polls
        ws.zero_()
        call(a)
        bad = assert_right_or_nan(out, lse, want, want_lse)
        assert (bad > 0) == (status() == abi.TR_ERR_TIMEOUT)
    a.wait_polls = 1  # the first loads cannot be there yet
    ws.zero_()
    call(a)
    assert status() == abi.TR_ERR_TIMEOUT
    assert assert_right_or_nan(out, lse, want, want_lse) > 0
    a.wait_polls = 0
    call(a)
    call(b)
    assert out.isnan().all() and lse.isnan().all() and few_out.isnan().all()
    assert status() == abi.TR_ERR_TIMEOUT
    abi.check(abi.lib().tr_workspace_clear(ctypes.c_void_p(ws.data_ptr()),
                                           abi.TR_ATTENTION_STATE_BYTES, ctypes.c_void_p(stream)),
              "tr_workspace_clear")
    call(a)
    call(b)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(few_out, few_want)
    assert status() == abi.TR_OK and not ws[:abi.TR_ATTENTION_STATE_BYTES].any()


def binding_timeouts(raises):
    args = long_chunks()
    want, want_lse = trb.paged_attention(*args, return_lse=True)
    assert trb.attention_status() == abi.TR_OK
    trb.set_attention_wait_limit(1)
    if raises:
        with pytest.raises(RuntimeError, match="timed out"):
            trb.paged_attention(*args)
    else:
        got = trb.paged_attention(*args, return_lse=True)
        assert assert_right_or_nan(*got, want, want_lse) > 0
    trb.set_attention_wait_limit(0)
    if not raises:
        assert trb.paged_attention(*args).isnan().all()
        assert trb.attention_status(reset=False) == abi.TR_ERR_TIMEOUT
        with torch.cuda.stream(torch.cuda.Stream()):
            assert trb.attention_status() == abi.TR_OK
            assert torch.equal(trb.paged_attention(*args), want)
            torch.cuda.current_stream().synchronize()
        assert trb.attention_status() == abi.TR_ERR_TIMEOUT
    assert trb.attention_status() == abi.TR_OK
    assert torch.equal(trb.paged_attention(*args), want)


@gpu
@pytest.mark.parametrize("raises", [False, True])
def test_attention_timeout_through_the_binding(raises):
    in_fresh_process(f"binding_timeouts({raises})", TRR_CHECK_STATUS=str(int(raises)))


# ---------------------------------------------------------------------------- the example
@gpu
def test_decoder_draws_no_token_for_idle_and_refused_requests():
    ex = load_example()
    model = ex.Decoder(ex.Shape(), 4, pages=8, longest=160)
    ints = dict(dtype=torch.int32, device=DEV)
    noise = torch.empty(4, model.shape.vocab, device=DEV).exponential_(generator=gen(3))
    heat = torch.ones(4, device=DEV)
    new = [20, 0, 140, 33]  # the third needs nine pages of eight, the fourth comes after it
    ids = model.step(torch.arange(sum(new), device=DEV), torch.tensor(new, **ints), noise, heat)
    assert int(ids[0]) >= 0 and ids[1:].tolist() == [-1, -1, -1]
    assert model.lens.tolist() == [20, 0, 0, 0]


# ---------------------------------------------------------------------------------- norms
@gpu
@pytest.mark.parametrize("width", [33, 768, 1000, 1920, 4096, 5001, 14336, 32760])
@pytest.mark.parametrize("eps", [1e-5, 1e-12])
def test_layer_norm_of_rows_of_one_value(width, eps):
    """Nothing is left but the bias.  The mean is off by c 2^-22 at most (a tree of sums) and the
    mean of the differences by 2^-20 of that, times 1 / sqrt(eps)."""
    for size in (1.0, 1e4, 1e6):
        c = torch.rand(300, generator=gen(width), device=DEV) * size
        h = c[:, None].expand(300, width).contiguous()
        h[0, 0] = math.nan
        w, b = torch.ones(width, device=DEV), torch.full((width,), 0.25, device=DEV)
        x = trb.residual_norm(None, h, pre=w, pre_bias=b, kind="layer", eps=eps)[1]
        assert x[0].isnan().all()
        assert float((x[1:] - 0.25).abs().max()) <= 1e-6 + size * 2.0 ** -42 / eps ** 0.5


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


@gpu
@pytest.mark.parametrize("vocab,dtype", [(5000, torch.float32), (4999, torch.bfloat16),
                                         (60001, torch.float32), (900001, torch.bfloat16)])
def test_sample_infinite_temperature(vocab, dtype):
    """Every finite logit has the same probability, -inf has none, +inf has all."""
    logits, noise = sample_inputs(3, vocab, dtype, vocab)
    logits[1, ::3] = -math.inf
    logits[2, 5:40:7] = math.inf
    heat = torch.full((3,), math.inf, device=DEV)
    ids, logprobs = trb.sample_tokens(logits, noise, heat)
    drawn = [logits[0] == logits[0], logits[1] > -math.inf, logits[2] == math.inf]
    for r, shares in enumerate(drawn):
        assert int(ids[r]) == int(torch.where(shares, noise[r].double(), math.inf).argmin())
        n = int(shares.sum())
        assert abs(float(logprobs[r]) + math.log(n)) <= 2e-5 * max(1.0, math.log(n))
    for k in (1, 20, 700):
        ids = trb.sample_tokens(logits, noise, heat, top_k=i32([k] * 3))[0]
        half = trb.sample_tokens(logits, noise, heat, top_k=i32([2 * k] * 3),
                                 top_p=torch.full((3,), 0.5, device=DEV))[0]
        for r in (0, 1):
            kept = np.argsort(-f64(logits[r]), kind="stable")[:k]
            assert int(ids[r]) == int(half[r]) == int(kept[np.argmin(f64(noise[r])[kept])])
    least = trb.sample_tokens(logits, noise, heat, min_p=torch.full((3,), 0.9, device=DEV))[0]
    assert torch.equal(least, trb.sample_tokens(logits, noise, heat)[0])


@gpu
@pytest.mark.parametrize("vocab,dtype", [(5000, torch.float32), (4999, torch.bfloat16),
                                         (900001, torch.bfloat16)])
@pytest.mark.parametrize("temperature", [1e-36, 1e-38, 1e-45])
def test_sample_temperatures_at_which_t_passes_fp32(vocab, dtype, temperature):
    """The greatest logit has all the probability (shared among its equals)."""
    logits, noise = sample_inputs(3, vocab, dtype, vocab)
    logits[2] -= 100
    heat = torch.full((3,), temperature, device=DEV)
    least = torch.full((3,), 0.1, device=DEV)
    for limits in (dict(), dict(top_k=i32([5] * 3)), dict(min_p=least), dict(top_p=least)):
        ids, logprobs = trb.sample_tokens(logits, noise, heat, **limits)
        for r in range(3):
            top = logits[r] == logits[r].max()
            assert int(ids[r]) == int(torch.where(top, noise[r].double(), math.inf).argmin()) \
                or "top_p" in limits and bool(top[ids[r]])
            assert abs(float(logprobs[r]) + math.log(int(top.sum()))) <= 2e-5


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [-3e4, 3e4])
def test_sample_min_p_of_logits_far_from_zero(shift, dtype):
    """The search's lower bound is rounded at the size of the logits, not of their differences."""
    logits, noise = sample_inputs(4, 20000, dtype, 11, scale=300.0)
    logits += shift
    heat = torch.tensor([0.01, 1.0, 40.0, 300.0], device=DEV)
    least = torch.tensor([0.5, 0.01, 0.3, 0.05], device=DEV)
    check_sample(logits, noise, heat, min_p=least)
