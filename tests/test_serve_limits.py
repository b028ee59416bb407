"""The serving operators at their limits: paths that ordinary inputs seldom reach, workspaces and
bounded waits through the C ABI, and the registered torch ops."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kernel_task_b200 as trb
from kernel_task_b200 import abi, library  # noqa: F401  (library registers the torch ops)
from oracle import serve_oracle as so
from test_serve import attention_case, check_attention, check_sample, i32

gpu = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------- sampling
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [3000, 40001])
def test_sample_draws_that_are_never_kept(vocab, dtype):
    # noise that turns the order round: every draw is the least likely token left, so the cut
    # itself has to be found
    g = torch.Generator(device=DEV).manual_seed(vocab)
    logits = torch.randn(6, vocab, generator=g, device=DEV).to(dtype)
    noise = torch.exp(2 * logits.float())
    ones = torch.ones(6, device=DEV)
    p = torch.tensor([0.9, 0.5, 0.999, 0.3, 0.7, 0.95], device=DEV)
    check_sample(logits, noise, ones, top_p=p)
    check_sample(logits, noise, ones, top_k=i32([700, 2000, 1500, 2999, 600, 1]))
    check_sample(logits, noise, ones, top_k=i32([700, 2000, 1500, 2999, 600, 1]), top_p=p,
                 min_p=torch.full((6,), 0.01, device=DEV))


@gpu
def test_sample_cut_inside_many_ties():
    # 20000 tokens of two values: the cut is a place among equals
    V = 20000
    logits = torch.zeros(3, V, device=DEV, dtype=torch.bfloat16)
    logits[:, ::2] = 1.0
    noise = torch.full((3, V), 1.0, device=DEV)
    ids = torch.arange(V, device=DEV)
    upper, lower = ids[::2], ids[1::2]
    k = 13000                                   # all of the upper, 3000 of the lower
    last = int(lower[2999])
    noise[0, last], noise[0, last + 2] = 1e-6, 1e-9
    mass = math.e * 10000 + 10000
    p = (math.e * 5000.5) / mass                # the upper's first 5001
    noise[1, upper[5000]], noise[1, upper[5001]] = 1e-6, 1e-9
    p2 = (math.e * 10000 + 4000.5) / mass       # the lower's first 4001
    noise[2, lower[4000]], noise[2, lower[4001]] = 1e-6, 1e-9
    got = trb.sample_tokens(logits, noise, torch.ones(3, device=DEV), top_k=i32([k, 0, 0]),
                            top_p=torch.tensor([1.0, p, p2], device=DEV))[0].tolist()
    assert got == [last, int(upper[5000]), int(lower[4000])]


@gpu
def test_sample_vocabulary_past_the_cluster():
    V = 900001
    g = torch.Generator(device=DEV).manual_seed(5)
    logits = (torch.randn(3, V, generator=g, device=DEV) * 3).to(torch.bfloat16)
    noise = torch.empty(3, V, device=DEV).exponential_(generator=g)
    heat = torch.tensor([1.0, 0.0, 0.7], device=DEV)
    check_sample(logits, noise, heat)
    check_sample(logits, noise, heat, top_k=i32([40, 0, 3]))
    check_sample(logits, noise, heat, top_k=i32([40, 0, 300]), top_p=torch.full((3,), 0.9, device=DEV),
                 min_p=torch.full((3,), 0.02, device=DEV))


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_sample_extreme_values(scale):
    g = torch.Generator(device=DEV).manual_seed(7)
    logits = torch.randn(4, 5000, generator=g, device=DEV) * scale
    noise = torch.empty(4, 5000, device=DEV).exponential_(generator=g)
    ones = torch.ones(4, device=DEV)
    # next to nothing between the logits: a uniform draw; everything: the greatest
    for limits in (dict(), dict(top_k=i32([0, 10, 900, 4999])),
                   dict(top_p=torch.tensor([1.0, 0.5, 0.9, 0.01], device=DEV))):
        got = trb.sample_tokens(logits, noise, ones, **limits)[0]
        if scale > 1:
            assert torch.equal(got, logits.argmax(1))
        else:
            check_sample(logits, noise, ones, **limits)


# ------------------------------------------------------------------- attention, the C ABI
def attention_struct(args, out, lse=None, **over):
    q, kp, vp, tables, lens, starts = args
    a = abi.TrAttention(q=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                        k_pages=kp.data_ptr(), v_pages=vp.data_ptr(), tables=tables.data_ptr(),
                        table_stride=tables.stride(0), lens=lens.data_ptr(),
                        starts=starts.data_ptr(), out=out.data_ptr(),
                        lse=lse.data_ptr() if lse is not None else None, tokens=q.shape[0],
                        requests=lens.shape[0], pages=kp.shape[0], columns=tables.shape[1],
                        page_size=kp.shape[2], heads=q.shape[1], kv_heads=kp.shape[1],
                        head_dim=q.shape[2], dtype=abi.TR_BF16, scale=q.shape[2] ** -0.5)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def need_of(a):
    n = ctypes.c_size_t()
    abi.check(abi.lib().tr_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)), "bytes")
    return n.value


@gpu
@pytest.mark.parametrize("new", [1, 100])
def test_attention_workspace(new):
    args = attention_case([700, 400], [new, new], 4, 2, 128, 16, torch.bfloat16)
    want = trb.paged_attention(*args)
    out = torch.zeros_like(want)
    a = attention_struct(args, out)
    need, stream = need_of(a), torch.cuda.current_stream().cuda_stream
    # only the state has to be zero: the rest may hold anything
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    ws[:abi.TR_ATTENTION_STATE_BYTES] = 0
    call = abi.lib().tr_paged_attention
    p = ctypes.c_void_p
    assert call(ctypes.byref(a), p(ws.data_ptr()), need - 1, p(stream)) == abi.TR_ERR_WORKSPACE
    assert call(ctypes.byref(a), None, need, p(stream)) == abi.TR_ERR_WORKSPACE
    assert call(ctypes.byref(a), p(ws.data_ptr() + 4), need, p(stream)) == abi.TR_ERR_ALIGN
    for _ in range(3):
        out.zero_()
        assert call(ctypes.byref(a), p(ws.data_ptr()), need, p(stream)) == abi.TR_OK
        assert torch.equal(out, want)
    assert not ws[:abi.TR_ATTENTION_STATE_BYTES].any()
    assert abi.workspace_status(ws.data_ptr(), need, stream=stream) == abi.TR_OK


@gpu
def test_attention_one_workspace_for_calls_of_any_shape():
    cases = [attention_case([3000, 40], [1, 1], 8, 2, 128, 16, torch.bfloat16),
             attention_case([900, 300, 77], [300, 150, 9], 8, 1, 64, 64, torch.bfloat16),
             attention_case([50] * 40, [1] * 40, 32, 8, 64, 16, torch.bfloat16),
             attention_case([2000], [9], 4, 4, 128, 32, torch.bfloat16)]
    want = [trb.paged_attention(*c) for c in cases]
    outs = [torch.zeros_like(w) for w in want]
    structs = [attention_struct(c, o) for c, o in zip(cases, outs)]
    need, stream = max(map(need_of, structs)), torch.cuda.current_stream().cuda_stream
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)
    for order in ([0, 1, 2, 3], [3, 1, 0, 2], [2, 0, 1, 3]):
        for i in order:
            outs[i].zero_()
            abi.check(abi.lib().tr_paged_attention(ctypes.byref(structs[i]),
                                                   ctypes.c_void_p(ws.data_ptr()), need,
                                                   ctypes.c_void_p(stream)), "attention")
            assert torch.equal(outs[i], want[i])


@gpu
def test_attention_timeout_is_reported_and_cleared():
    args = attention_case([900, 700], [300, 200], 8, 2, 128, 16, torch.bfloat16)
    want = trb.paged_attention(*args)
    out = torch.zeros_like(want)
    a = attention_struct(args, out, wait_polls=1)
    need, stream = need_of(a), torch.cuda.current_stream().cuda_stream
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)
    ptr = ctypes.c_void_p(ws.data_ptr())
    # one poll a wait: the waits for the loads run out on a healthy GPU, and the kernel returns
    seen = set()
    for _ in range(3):
        ws.zero_()
        assert abi.lib().tr_paged_attention(ctypes.byref(a), ptr, need, ctypes.c_void_p(stream)) == abi.TR_OK
        seen.add(abi.workspace_status(ws.data_ptr(), need, stream=stream))
    assert seen <= {abi.TR_OK, abi.TR_ERR_TIMEOUT}
    # the state cleared, the next call is right
    abi.check(abi.lib().tr_workspace_clear(ptr, abi.TR_ATTENTION_STATE_BYTES, ctypes.c_void_p(stream)),
              "clear")
    a.wait_polls = 0
    abi.check(abi.lib().tr_paged_attention(ctypes.byref(a), ptr, need, ctypes.c_void_p(stream)), "call")
    assert torch.equal(out, want)
    assert abi.workspace_status(ws.data_ptr(), need, stream=stream) == abi.TR_OK


@gpu
def test_attention_starts_that_do_not_rise():
    # starts of a corrupt plan: no read or write outside the arrays; what rows hold is not said
    args = list(attention_case([40, 50, 60], [10, 20, 30], 4, 2, 64, 16, torch.bfloat16))
    for bad in ([0, 50, 20, 60], [-5, 10, 30, 90], [0, 2 ** 31 - 1, 3, 60], [70, 80, 90, 100]):
        args[5] = i32(bad)
        out = trb.paged_attention(*args)
        torch.cuda.synchronize()
        assert out.shape == args[0].shape
    args[5] = i32([0, 10, 30, 60])
    check_attention(tuple(args))


@gpu
@pytest.mark.parametrize("new", [1, 40])
def test_attention_many_requests(new):
    # more requests than a block has threads
    lens = [(7 * i) % 61 + new for i in range(600)]
    args = attention_case(lens, [new] * 600 if new == 1 else [new if i % 50 == 0 else 0 for i in range(600)],
                          2, 1, 64, 16, torch.bfloat16)
    check_attention(args)


# ------------------------------------------------------------------------- torch.library
def test_registered_ops_know_their_shapes():
    with FakeTensorMode():
        b16 = dict(dtype=torch.bfloat16)
        ints = dict(dtype=torch.int32)
        lens, tables, free = torch.empty(3, **ints), torch.empty(3, 4, **ints), torch.empty(9, **ints)
        plan = torch.ops.trring.plan_step(lens, lens, tables, free, free[:1], 16, 7)
        assert [t.shape[0] for t in plan] == [7, 7, 4, 3, 3, 1] and plan[0].dtype == torch.int64
        q, pool = torch.empty(5, 8, 64, **b16), torch.empty(9, 2, 16, 64, **b16)
        out, lse = torch.ops.trring.paged_attention(q, pool, pool, tables, lens, torch.empty(4, **ints))
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (5, 8) and lse.dtype == torch.float32
        k = torch.empty(5, 2, 64, **b16)
        assert torch.ops.trring.append_kv(k, k, pool, pool.clone(), torch.empty(5, dtype=torch.int64)) is None
        h, w = torch.empty(5, 32, **b16), torch.empty(32, **b16)
        got = torch.ops.trring.residual_norm(h.float(), h, w, w, None, None, None, "rms", 1e-6, 1.0, 1.0)
        assert all(t.shape == h.shape and t.dtype == h.dtype for t in got)
        lg = torch.empty(4, 99)
        ids, lp = torch.ops.trring.sample_tokens(lg, lg, lg[:, 0], None, None, None)
        assert ids.shape == (4,) and ids.dtype == torch.int64 and lp.dtype == torch.float32


@gpu
def test_registered_ops_run():
    args = attention_case([40, 9], [1, 9], 4, 2, 64, 16, torch.bfloat16)
    out, lse = torch.ops.trring.paged_attention(*args)
    want = trb.paged_attention(*args, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    lens, tables = i32([3, 0]), i32([[5, -1], [-1, -1]])
    got = torch.ops.trring.plan_step(lens, i32([1, 20]), tables, i32([1, 2, 3]), i32([3]), 16, 21)
    ref = so.plan_step([3, 0], [1, 20], np.array([[5, -1], [-1, -1]]), [1, 2, 3], 3, 16, 21)
    for t, r in zip(got[:5], ref[:5]):
        assert np.array_equal(t.cpu().numpy(), r)
    h = torch.randn(3, 64, device=DEV).bfloat16()
    w = torch.ones(64, device=DEV).bfloat16()
    a = torch.ops.trring.residual_norm(h, h, w, w, None, None, None, "rms", 1e-6, 1.0, 1.0)
    b = trb.residual_norm(h, h, post=w, pre=w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    lg, nz = torch.randn(2, 50, device=DEV), torch.rand(2, 50, device=DEV)
    one = torch.ones(2, device=DEV)
    assert torch.equal(torch.ops.trring.sample_tokens(lg, nz, one, None, None, None)[0],
                       trb.sample_tokens(lg, nz, one)[0])
