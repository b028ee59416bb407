"""The serving operators on the GPU against float64 numpy restatements, at the sizes, strides and
masks where they can go wrong.

Tolerances.  u is the unit of rounding of the output type, 2^-p for p significant bits: 2^-8 for
bf16, 2^-11 for fp16, 2^-24 for fp32.
  attention  out is rounded once (u |out|) and the probabilities that multiply V are rounded to
             the same type (u sum p|v|); scores are fp32 sums
             of exact products (relative 2^-22 of sums of magnitude below 100) and exp adds
             2^-21, together below 1e-4 of sum p|v|.  lse: 1e-4 absolute.
  norm       fp32 sums over at most 32768 terms in a tree: below 1e-5 of the row's norm-sized
             values, plus one rounding u |out|.
  sample     tokens equal where no decision is nearer than 1e-4 (fp32 errors of t, log and
             masses are below 2e-5), else equal to what a limit moved by that much gives;
             logprobs to 2e-5.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kernel_task_b200 as trb
from oracle import serve_oracle as so

gpu = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------ step plan
def make_pool(lens, page, columns, spare, seed=0):
    rng = np.random.default_rng(seed)
    counts = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(counts) + spare).astype(np.int32)
    tables = np.full((len(lens), columns), -1, np.int32)
    at = 0
    for r, n in enumerate(counts):
        tables[r, :n] = ids[at:at + n]
        at += n
    return tables, ids[at:].copy(), sum(counts) + spare


def check_plan(lens, new, page, columns, spare, tokens=None, free_count=None, inplace=False):
    tables, free, _ = make_pool([max(n, 0) for n in lens], page, columns, spare)
    fc = len(free) if free_count is None else free_count
    tokens = sum(max(n, 0) for n in new) if tokens is None else tokens
    want = so.plan_step(lens, new, tables, free, fc, page, tokens)
    d = dict(lens=i32(lens), tables=i32(tables), free=i32(free), count=i32([fc]))
    got = trb.plan_step(d["lens"], i32(new), d["tables"], d["free"], d["count"], page, tokens,
                        inplace=inplace)
    for name, w in zip(("slots", "positions", "starts", "lens", "granted"), want):
        assert np.array_equal(getattr(got, name).cpu().numpy(), w), name
    assert int(got.free_count) == want[5]
    assert np.array_equal(d["tables"].cpu().numpy(), want[6])
    assert np.array_equal(d["free"].cpu().numpy(), free)
    if inplace:
        assert got.lens.data_ptr() == d["lens"].data_ptr()
        assert got.free_count.data_ptr() == d["count"].data_ptr()
    else:
        assert d["lens"].cpu().tolist() == list(lens) and int(d["count"]) == fc
    return got


@gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_plan_ragged(page, inplace):
    rng = np.random.default_rng(page)
    lens = rng.integers(0, 300, 77).tolist()
    new = [int(n) for n in rng.integers(0, 50, 77)]
    check_plan(lens, new, page, 400 // page + 1, 4000, inplace=inplace)


@gpu
@pytest.mark.parametrize("requests", [1, 31, 1024, 1025, 5000])
def test_plan_many_requests(requests):
    rng = np.random.default_rng(requests)
    check_plan(rng.integers(0, 64, requests).tolist(), rng.integers(0, 3, requests).tolist(), 16,
               6, requests)


@gpu
def test_plan_one_long_prompt_on_a_cluster():
    check_plan([5, 0, 17], [3, 40001, 0], 32, 1300, 1300, tokens=40010)


@gpu
def test_plan_refusals_by_pool_columns_and_tokens():
    # the pool runs out at the third request; the fourth needs no page, the fifth one again
    check_plan([16, 30, 16, 3, 16], [1, 20, 100, 2, 1], 16, 20, 4)
    # the table is too narrow for the second
    check_plan([16, 30, 16], [1, 400, 1], 16, 8, 100)
    # the slot map ends inside the second
    check_plan([0, 0, 0], [10, 10, 10], 16, 8, 100, tokens=15)
    # nothing is free; padding past the last token
    check_plan([15, 16, 0], [1, 1, 0], 16, 8, 0, tokens=9)
    check_plan([15, 16], [1, 1], 16, 8, 5, free_count=0)


@gpu
def test_plan_empty_and_idle():
    check_plan([], [], 16, 4, 3)
    check_plan([], [], 16, 4, 3, tokens=7)
    check_plan([0, 0], [0, 0], 16, 4, 3)
    check_plan([4, 9], [-3, 2], 16, 4, 3)   # a negative count is none


@gpu
def test_release_and_reuse():
    page, lens = 16, [40, 0, 16, 17, 100]
    tables, free, _ = make_pool(lens, page, 9, 5)
    pool = np.full(len(free) + 40, -7, np.int32)
    pool[:len(free)] = free
    d = dict(lens=i32(lens), tables=i32(tables), free=i32(pool), count=i32([len(free)]))
    trb.release_pages(d["lens"], i32([1, 1, 0, 1, 0]), d["tables"], d["free"], d["count"], page)
    back = list(tables[0, :3]) + list(tables[3, :2])
    assert d["lens"].cpu().tolist() == [0, 0, 16, 0, 100]
    assert int(d["count"]) == len(free) + 5
    assert d["free"].cpu().tolist()[:len(free) + 5] == list(free) + back
    assert (d["tables"].cpu().numpy()[[0, 1, 3]] == -1).all()
    assert np.array_equal(d["tables"].cpu().numpy()[[2, 4]], tables[[2, 4]])
    step = trb.plan_step(d["lens"], i32([33, 0, 0, 0, 0]), d["tables"], d["free"], d["count"], page,
                         33)
    assert d["tables"].cpu().tolist()[0][:3] == back[::-1][:3]
    assert int(step.free_count) == len(free) + 2


@gpu
def test_release_large():
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 900, 1500).tolist()
    tables, free, total = make_pool(lens, 16, 60, 11)
    pool = np.full(total, -1, np.int32)
    pool[:11] = free
    done = rng.integers(0, 2, 1500)
    d = dict(lens=i32(lens), tables=i32(tables), free=i32(pool), count=i32([11]))
    trb.release_pages(d["lens"], i32(done), d["tables"], d["free"], d["count"], 16)
    back = [p for r in range(1500) if done[r] for p in tables[r, :-(-lens[r] // 16)]]
    assert d["free"].cpu().tolist()[:11 + len(back)] == list(free) + back
    assert int(d["count"]) == 11 + len(back)


# --------------------------------------------------------------------------------- append
@gpu
@pytest.mark.parametrize("dtype,source", [(torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float32),
                                          (torch.float32, torch.float32)])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 8, 1), (5, 8, 128, 16), (77, 3, 64, 7),
                                                   (33, 2, 20, 16)])
def test_append(dtype, source, tokens, heads, dim, page):
    g = gen(tokens)
    both = torch.randn(tokens, 2 * heads * dim, generator=g, device=DEV).to(source)
    k = both[:, :heads * dim].unflatten(1, (heads, dim))
    v = both[:, heads * dim:].unflatten(1, (heads, dim))
    pages = tokens // page + 4
    shape = (pages, heads, page, dim)
    kp = torch.randn(shape, generator=g, device=DEV).to(dtype)
    vp = torch.randn(shape, generator=g, device=DEV).to(dtype)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    if tokens > 2:
        slots[1] = -1
        slots[2] = pages * page      # past the pools: skipped
    want_k, want_v = kp.clone(), vp.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, :, s % page] = k[t].to(dtype)
            want_v[s // page, :, s % page] = v[t].to(dtype)
    trb.append_kv(k, v, kp, vp, slots)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


@gpu
def test_append_strides_and_alignment():
    base = torch.randn(9, 3, 2, 17, device=DEV).to(torch.bfloat16)
    k = base[:, :, 0, 1:].transpose(0, 1)       # [3, 9, 16], odd strides and offset
    v = base[:, :, 1, :16].transpose(0, 1)
    kp = torch.zeros(2, 9, 4, 16, device=DEV, dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    slots = torch.tensor([6, 0, 3], device=DEV)
    trb.append_kv(k, v, kp, vp, slots)
    for t, s in enumerate([6, 0, 3]):
        assert torch.equal(kp[s // 4, :, s % 4], k[t]) and torch.equal(vp[s // 4, :, s % 4], v[t])
    trb.append_kv(k[:, :, ::2], v[:, :, ::2], torch.zeros(2, 9, 4, 8, device=DEV).to(k.dtype),
                  torch.zeros(2, 9, 4, 8, device=DEV).to(k.dtype), slots)
    trb.append_kv(k[:0], v[:0], kp, vp, slots[:0])


# ------------------------------------------------------------------------------ attention
def attention_case(lens, new, heads, kv_heads, dim, page, dtype, seed=0, dirty=True):
    """Inputs with a shuffled pool whose unused rows hold NaN (and Inf), as a pool may."""
    g = gen(seed)
    tables, _, total = make_pool(lens, page, max([-(-n // page) for n in lens] + [1]) + 1, 2, seed)
    shape = (total, kv_heads, page, dim)
    kp = torch.randn(shape, generator=g, device=DEV).to(dtype)
    vp = torch.randn(shape, generator=g, device=DEV).to(dtype)
    if dirty:
        used = torch.zeros(total, page, dtype=torch.bool)
        for r, n in enumerate(lens):
            for j in range(n):
                used[int(tables[r, j // page]), j % page] = True
        mask = ~used[:, None, :, None].to(DEV)
        kp.masked_fill_(mask, math.nan)
        vp.masked_fill_(mask, math.inf)
    both = torch.randn(sum(new), (heads + 2 * kv_heads) * dim, generator=g, device=DEV).to(dtype)
    q = both[:, :heads * dim].unflatten(1, (heads, dim))
    starts = np.concatenate([[0], np.cumsum(new)])
    return q, kp, vp, i32(tables), i32(lens), i32(starts)


def check_attention(args, scale=None):
    q, kp, vp, tables, lens, starts = args
    out, lse = trb.paged_attention(*args, scale=scale, return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:2]
    ref, ref_lse, spread = so.paged_attention(
        f64(q), f64(kp), f64(vp), tables.cpu().numpy(), lens.cpu().numpy(), starts.cpu().numpy(),
        q.shape[2] ** -0.5 if scale is None else scale)
    u = UNIT[q.dtype]
    bound = u * np.abs(ref) + (u + 1e-4) * spread + 1e-30
    err = np.abs(f64(out) - ref)
    assert np.isfinite(f64(out)).all()
    assert (err <= bound).all(), (err / bound).max()
    got_lse = f64(lse)
    none = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(got_lse), none)
    assert (f64(out)[none] == 0).all()
    assert np.abs(got_lse[~none] - ref_lse[~none]).max(initial=0.0) <= 1e-4
    # the same bits again, and without the log-sums
    again = trb.paged_attention(*args, scale=scale)
    assert torch.equal(again, out)
    return out


LAYOUTS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (14, 2, 64), (8, 1, 128), (32, 8, 64), (20, 1, 64)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_attention_single_tokens(heads, kv_heads, dim, dtype):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 200, 1]
    check_attention(attention_case(lens, [1] * len(lens), heads, kv_heads, dim, 16, dtype))


@gpu
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 128, 512])
def test_attention_page_sizes(page):
    lens = [1, 130, 64, 257]
    check_attention(attention_case(lens, [1] * 4, 8, 2, 64, page, torch.bfloat16))
    check_attention(attention_case(lens, [1, 100, 33, 7], 8, 2, 64, page, torch.bfloat16))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_attention_chunks(heads, kv_heads, dim, dtype):
    lens, new = [70, 5, 131, 129, 260], [70, 1, 33, 129, 2]
    check_attention(attention_case(lens, new, heads, kv_heads, dim, 16, dtype))


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (2, 2, 64)])
def test_attention_long_chunks(heads, kv_heads, dim):
    lens, new = [400, 900, 311], [400, 300, 1]
    check_attention(attention_case(lens, new, heads, kv_heads, dim, 32, torch.bfloat16))


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 1, 64)])
def test_attention_long_context_is_split(heads, kv_heads, dim):
    lens = [5000, 1, 3333]
    check_attention(attention_case(lens, [1, 1, 1], heads, kv_heads, dim, 64, torch.bfloat16))
    check_attention(attention_case([5000, 2100], [3, 40], heads, kv_heads, dim, 64, torch.float16))


@gpu
@pytest.mark.parametrize("dim", [8, 40, 80, 96, 192, 256])
def test_attention_general_kernel(dim):
    for dtype in (torch.bfloat16, torch.float32):
        check_attention(attention_case([1, 40, 65], [1, 3, 65], 4, 2, dim, 16, dtype))


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_rows_that_see_nothing(dim):
    # idle requests, requests without a cache, and more tokens than are cached
    for dtype in (torch.bfloat16, torch.float32):
        args = list(attention_case([0, 20, 7, 0, 33], [1, 0, 9, 5, 1], 4, 2, dim, 16, dtype))
        check_attention(args)
    args[4] = i32([0, 0, 0, 0, 0])
    assert not trb.paged_attention(*args).any()
    args[4] = i32([-4, 20, -1, 0, 33])
    check_attention(args)


@gpu
@pytest.mark.parametrize("new", [[1, 1], [50, 40]])
def test_attention_tokens_outside_all_requests(new):
    q, kp, vp, tables, lens, starts = attention_case([64, 80], new, 4, 2, 64, 16, torch.bfloat16)
    pad = torch.randn(6, 4, 64, device=DEV).to(q.dtype)
    padded = torch.cat([pad[:2], q, pad[2:]])
    out, lse = trb.paged_attention(padded, kp, vp, tables, lens, starts + 2, return_lse=True)
    want, want_lse = trb.paged_attention(q, kp, vp, tables, lens, starts, return_lse=True)
    n = q.shape[0]
    assert torch.equal(out[2:n + 2], want) and torch.equal(lse[2:n + 2], want_lse)
    assert not out[:2].any() and not out[n + 2:].any()
    assert (lse[:2] == -math.inf).all() and (lse[n + 2:] == -math.inf).all()


@gpu
@pytest.mark.parametrize("new", [1, 60])
def test_attention_bad_page_ids_read_as_zeros(new):
    q, kp, vp, tables, lens, starts = attention_case([100], [new], 4, 2, 64, 16, torch.bfloat16)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        tables[0, 2] = bad
        check_attention((q, kp, vp, tables, lens, starts))


@gpu
@pytest.mark.parametrize("new", [1, 60])
def test_attention_large_scores_and_scale(new):
    q, kp, vp, tables, lens, starts = attention_case([90], [new], 4, 2, 64, 16, torch.bfloat16)
    # scores of several hundred: the running maximum has to move, sums must not overflow
    kp.mul_(torch.linspace(1, 30, 16, device=DEV)[None, None, :, None])
    got = trb.paged_attention(q, kp, vp, tables, lens, starts, scale=1.0)
    ref, _, spread = so.paged_attention(f64(q), f64(kp), f64(vp), tables.cpu().numpy(),
                                        lens.cpu().numpy(), starts.cpu().numpy(), 1.0)
    # scores up to ~1000: their fp32 error 1000 * 2^-20 is what p is off by
    assert (np.abs(f64(got) - ref) <= 2 ** -8 * np.abs(ref) + 2 ** -7 * spread).all()
    check_attention(attention_case([90], [new], 4, 2, 64, 16, torch.bfloat16), scale=0.01)


@gpu
def test_attention_unaligned_and_strided_queries():
    q, *rest = attention_case([64, 33], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    want = trb.paged_attention(q.contiguous(), *rest)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=q.dtype)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(trb.paged_attention(odd, *rest), want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(trb.paged_attention(turned, *rest), want)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, :rest[2].shape[1]] = rest[2]
    rest[2] = wide[:, :rest[2].shape[1]]
    assert torch.equal(trb.paged_attention(q, *rest), want)
    assert trb.paged_attention(q[:0], *rest[:4], i32([0, 0, 0])).shape == (0, 4, 64)


@gpu
def test_attention_offsets_past_32_bits():
    # a pool of more than 2^31 elements: the last page is past what 32 bits address
    pages, page, dim = 17000, 1024, 128
    kp = torch.zeros(pages, 1, page, dim, device=DEV, dtype=torch.float16)
    vp = torch.zeros_like(kp)
    g = gen(1)
    k = torch.randn(1024, 1, dim, generator=g, device=DEV).half()
    v = torch.randn(1024, 1, dim, generator=g, device=DEV).half()
    slots = torch.arange(1024, device=DEV) + (pages - 1) * page
    trb.append_kv(k, v, kp, vp, slots)
    assert torch.equal(kp[-1, 0], k[:, 0])
    for new in (1, 200):
        q = torch.randn(new, 4, dim, generator=g, device=DEV).half()
        rest = (i32([1000]), i32([0, new]))
        far = trb.paged_attention(q, kp, vp, i32([[pages - 1]]), *rest)
        near = trb.paged_attention(q, kp[-1:].clone(), vp[-1:].clone(), i32([[0]]), *rest)
        assert torch.equal(far, near)


@gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 70, 5]])
def test_attention_on_two_streams_and_in_a_graph(new):
    args = attention_case([3000, 2500, 700], new, 8, 2, 128, 16, torch.bfloat16)
    want = trb.paged_attention(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(trb.paged_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = trb.paged_attention(*args)
    for _ in range(3):
        captured.zero_()
        graph.replay()
        assert torch.equal(trb.paged_attention(*args), want)
        torch.cuda.synchronize()
        assert torch.equal(captured, want)


# ---------------------------------------------------------------------------------- norms
def check_norm(T, W, dtype, kind="rms", y_dtype=None, gate="channel", post=True, pre=True,
               bias=False, with_y=True, seed=0, eps=1e-5, scales=(1.0, 0.5), shift=0.0):
    g = gen(seed)

    def rand(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(to)

    y = (rand(T, W, scale=3.0, to=torch.float32) + shift).to(y_dtype or dtype) if with_y else None
    h = rand(T, W, scale=2.0)
    gt = {"none": None, "channel": rand(W), "token": rand(T, W)}[gate] if with_y else None
    p = dict(post=1 + rand(W, scale=0.1) if post and with_y else None,
             pre=1 + rand(W, scale=0.1) if pre else None,
             post_bias=rand(W, scale=0.1) if bias and post and with_y else None,
             pre_bias=rand(W, scale=0.1) if bias and pre else None)
    got = trb.residual_norm(y, h, gate=gt, kind=kind, eps=eps, residual_scale=scales[0],
                            branch_scale=scales[1], **p)
    want = so.residual_norm(f64(y), f64(h), gate=f64(gt), kind=kind, eps=eps,
                            residual_scale=scales[0], branch_scale=scales[1],
                            **{n: f64(t) for n, t in p.items()})
    u = UNIT[dtype]
    size = max(1.0, np.abs(want[0]).max(initial=0.0))
    assert np.abs(f64(got[0]) - want[0]).max(initial=0.0) <= u * size + 1e-5 * size
    if pre:
        size = max(1.0, np.abs(want[1]).max(initial=0.0))
        assert (np.abs(f64(got[1]) - want[1]) <= u * np.abs(want[1]) + 1e-5 * size).all()
    else:
        assert got[1] is None
    return got


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [1, 7, 8, 33, 256, 264, 512, 520, 1000, 1920, 2048, 2056, 2880,
                                   4096, 4104, 8192, 8200, 14336, 16392, 32768])
def test_norm_widths(width, kind):
    check_norm(3, width, torch.bfloat16, kind, bias=kind == "layer")
    check_norm(3, width, torch.float16, kind, y_dtype=torch.float32, gate="token")


@gpu
@pytest.mark.parametrize("width", [33, 250, 2001, 5001, 9001, 32767])
def test_norm_widths_without_vectors(width):
    check_norm(5, width, torch.float16, "layer", gate="token", bias=True)
    check_norm(2, width, torch.float32, "rms")


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 9, 1000, 5001])
def test_norm_tokens(tokens):
    check_norm(tokens, 256, torch.bfloat16, gate="token")
    check_norm(tokens, 1024, torch.bfloat16, "layer", y_dtype=torch.float32)


@gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("post,pre,bias,with_y", [(True, True, True, True), (False, True, False, True),
                                                  (True, False, True, True), (False, False, False, True),
                                                  (False, True, True, False)])
def test_norm_parts(post, pre, bias, with_y, gate):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        check_norm(4, 640, dtype, "layer", gate=gate, post=post, pre=pre, bias=bias, with_y=with_y)
        check_norm(4, 640, dtype, "rms", gate=gate, post=post, pre=pre, bias=bias, with_y=with_y,
                   scales=(0.7, -1.5))


@gpu
def test_norm_large_mean_and_zero_rows():
    # a mean 3000 times the spread: sums of squares about zero would lose the variance
    check_norm(3, 2048, torch.bfloat16, "layer", y_dtype=torch.float32, shift=1e4)
    z = torch.zeros(2, 512, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    h, x = trb.residual_norm(z, z, post=w, pre=w, eps=1e-6)
    assert not h.any() and not x.any()


@gpu
def test_norm_strides_and_alignment():
    g = gen(4)
    big = torch.randn(6, 4, 520, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(512, generator=g, device=DEV).to(torch.bfloat16)
    want = trb.residual_norm(big[:, 1, :512].contiguous(), big[:, 0, :512].contiguous(), post=w, pre=w,
                             gate=big[:, 2, :512].contiguous())
    got = trb.residual_norm(big[:, 1, :512], big[:, 0, :512], post=w, pre=w, gate=big[:, 2, :512])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # rows that start off a 16-byte boundary, and columns that are not contiguous
    for cut in (slice(1, 513), slice(0, 1024, 2)):
        wide = torch.randn(6, 1030, generator=g, device=DEV).to(torch.bfloat16)
        a, b = wide[:, cut], big[:, 0, :512]
        got = trb.residual_norm(a, b, post=w, pre=w)
        want = trb.residual_norm(a.contiguous(), b.contiguous(), post=w, pre=w)
        for x, y in zip(got, want):
            torch.testing.assert_close(x, y, rtol=2 ** -7, atol=1e-5)
    assert trb.residual_norm(big[:0, 1, :512], big[:0, 0, :512], pre=w)[1].shape == (0, 512)


# --------------------------------------------------------------------------------- sampling
def second_best(logits, noise, temperature, token):
    """Tokens whose t - log(noise) is within 1e-4 of the drawn one's, with their logprobs."""
    t = np.where(np.isnan(logits), -np.inf, logits) / (temperature if temperature > 0 else 1.0)
    key = t - np.log(noise)
    z = np.log(np.exp(t - t.max()).sum()) + t.max()
    return [(int(i), t[i] - z) for i in np.flatnonzero(np.abs(key - key[token]) <= 1e-4)]


def check_sample(logits, noise, temperature, top_k=None, top_p=None, min_p=None):
    got, logprobs = trb.sample_tokens(logits, noise, temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    l, n = f64(logits), f64(noise)
    for r in range(l.shape[0]):
        k, p, m = (float(x[r]) if x is not None else d
                   for x, d in ((top_k, 0), (top_p, 1.0), (min_p, 0.0)))
        token, logprob, clear = so.sample(l[r], n[r], float(temperature[r]), int(k), p, m, 1e-4)
        if not clear:
            near = [so.sample(l[r], n[r], float(temperature[r]), int(k), p * (1 + a) if p < 1 else p,
                              m * (1 + b), 0.0)
                    for a in (0, -3e-4, 3e-4) for b in (0, -2e-4, 2e-4)]
            near += second_best(l[r], n[r], float(temperature[r]), token)
            match = [e for e in near if e[0] == int(got[r])]
            assert match, (r, int(got[r]), token)
            token, logprob = match[0][:2]
        assert int(got[r]) == token, (r, int(got[r]), token)
        if token < 0:
            assert float(logprobs[r]) == -math.inf
        else:
            assert abs(float(logprobs[r]) - logprob) <= 2e-5 * max(1.0, abs(logprob)), r
    return got


def sample_inputs(R, V, dtype, seed, scale=2.5):
    g = gen(seed)
    logits = (torch.randn(R, V, generator=g, device=DEV) * scale).to(dtype)
    return logits, torch.empty(R, V, device=DEV).exponential_(generator=g)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1024, 4099, 50021, 131072, 200003])
def test_sample_vocabularies(vocab, dtype):
    R = 12
    logits, noise = sample_inputs(R, vocab, dtype, vocab)
    heat = torch.tensor([0, 0.5, 1, 1.5] * 3, device=DEV)
    k = i32([0, 1, 5, 50, 300, 1000] * 2)
    p = torch.tensor([1, 0.9, 0.5, 0.99, 0.1, 0.75], device=DEV).repeat(2)
    m = torch.tensor([0, 0.1, 0.02, 0], device=DEV).repeat(3)
    check_sample(logits, noise, heat)
    check_sample(logits, noise, heat, top_k=k)
    check_sample(logits, noise, heat, top_p=p)
    check_sample(logits, noise, heat, min_p=m)
    check_sample(logits, noise, heat, top_k=k, top_p=p, min_p=m)


@gpu
def test_sample_flat_and_peaked_rows():
    logits, noise = sample_inputs(8, 3001, torch.bfloat16, 1)
    heat = torch.ones(8, device=DEV)
    for flat in (torch.zeros_like(logits), torch.full_like(logits, -3.0)):
        # all tied: the first k, and of those the first half, by index
        got = check_sample(flat, noise, heat, top_k=i32([100] * 8))
        assert (got < 100).all()
        got = check_sample(flat, noise, heat, top_k=i32([100] * 8),
                           top_p=torch.full((8,), 0.495, device=DEV))
        assert (got < 50).all()
        got = trb.sample_tokens(flat, noise, torch.zeros(8, device=DEV))[0]
        assert not got.any()
    logits[:, 17] = 100.0
    got = check_sample(logits, noise, heat, top_p=torch.full((8,), 0.9, device=DEV))
    assert (got == 17).all()


@gpu
def test_sample_ties_at_the_cut_go_to_the_lower_index():
    V = 5000
    logits = torch.full((1, V), -1.0, device=DEV)
    logits[0, 4000:4010] = 2.0
    logits[0, 100:4000:13] = 1.0                 # 300 ties
    tied = list(range(100, 4000, 13))
    noise = torch.full((1, V), 1.0, device=DEV)
    for k, last in ((11, tied[0]), (60, tied[49]), (310, tied[299])):
        n = noise.clone()
        n[0, last] = 1e-6                         # the last tie kept wins
        if last + 13 < 4000:
            n[0, last + 13] = 1e-9                # the first one dropped would have
        got = trb.sample_tokens(logits, n, torch.ones(1, device=DEV), top_k=i32([k]))[0]
        assert int(got) == last
    # equal keys everywhere: the lowest index of the greatest
    got = trb.sample_tokens(logits, noise, torch.ones(1, device=DEV))[0]
    assert int(got) == 4000


@gpu
def test_sample_masks_infinities_and_nan():
    logits, noise = sample_inputs(9, 2000, torch.float32, 2)
    low = torch.finfo(torch.float32).min
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 5:] = -math.inf
    logits[3] = low
    logits[4, 7:] = low
    logits[5, ::2] = math.nan
    logits[6] = -math.inf
    logits[6, 1234] = -5.0
    logits[7, 40] = math.inf
    logits[7, 90] = math.inf
    logits[8, :] = -0.0
    logits[8, 3] = 0.0
    heat = torch.ones(9, device=DEV)
    for k, p in ((0, 1.0), (3, 1.0), (0, 0.9), (3, 0.9)):
        got = trb.sample_tokens(logits, noise, heat, top_k=i32([k] * 9),
                                top_p=torch.full((9,), p, device=DEV))
        ids, lp = got[0].tolist(), got[1].tolist()
        assert ids[0] == -1 and ids[1] == -1 and lp[0] == lp[1] == -math.inf
        assert ids[2] < 5 and ids[4] < 7 and ids[5] % 2 == 1 and ids[6] == 1234 and ids[7] in (40, 90)
        assert abs(lp[6]) < 1e-6 and abs(lp[7] + math.log(2)) < 1e-6
        assert 0 <= ids[3] < 2000 and abs(lp[3] + math.log(2000)) < 1e-4
        assert abs(lp[8] + math.log(2000)) < 1e-4
    got = trb.sample_tokens(logits, noise, torch.zeros(9, device=DEV))[0].tolist()
    assert got[:2] == [-1, -1] and got[3] == 0 and got[7] == 40 and got[8] == 0


@gpu
def test_sample_limits_out_of_range():
    logits, noise = sample_inputs(4, 3000, torch.bfloat16, 3)
    heat = torch.tensor([1.0, -1.0, math.nan, 0.7], device=DEV)
    best = logits.float().argmax(1)
    got = trb.sample_tokens(logits, noise, heat)[0]
    assert got[1] == best[1] and got[2] == best[2]      # not above 0: greedy
    free = trb.sample_tokens(logits, noise, torch.ones(4, device=DEV))[0]
    ones = torch.ones(4, device=DEV)
    same = trb.sample_tokens(logits, noise, ones, top_k=i32([-1, 3000, 9999, 0]), top_p=ones * 3,
                             min_p=-ones)[0]
    assert torch.equal(free, same)
    # nothing would be left: the greatest always is
    top = torch.where(logits.float() == logits.float().amax(1, keepdim=True))
    for limits in (dict(top_p=ones * 0), dict(min_p=ones * 7), dict(top_k=i32([1] * 4))):
        got = trb.sample_tokens(logits, noise, ones, **limits)[0].tolist()
        for r in range(4):
            assert got[r] in top[1][top[0] == r].tolist()
    assert trb.sample_tokens(logits[:0], noise[:0], heat[:0])[0].shape == (0,)


@gpu
def test_sample_strided_rows():
    big, noise = sample_inputs(7, 4003, torch.bfloat16, 5)
    wide = torch.empty(7, 4003, device=DEV).exponential_(generator=gen(6))
    for a, b in ((1, 4001), (3, 2000), (0, 4003)):
        heat = torch.full((7,), 0.9, device=DEV)
        k, p = i32([40] * 7), torch.full((7,), 0.95, device=DEV)
        got = trb.sample_tokens(big[:, a:b], wide[:, a:b], heat, top_k=k, top_p=p)
        want = trb.sample_tokens(big[:, a:b].contiguous(), wide[:, a:b].contiguous(), heat, top_k=k,
                                 top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_sample_draws_with_the_probabilities():
    # 20000 draws of a small distribution: each count within 5 standard deviations of n p
    n, V = 20000, 11
    logits = torch.linspace(-1, 1, V, device=DEV).repeat(n, 1)
    noise = torch.empty(n, V, device=DEV).exponential_(generator=gen(8))
    ids = trb.sample_tokens(logits, noise, torch.ones(n, device=DEV))[0]
    p = torch.softmax(logits[0].double(), 0)
    count = torch.bincount(ids, minlength=V).double()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


# ------------------------------------------------------------------------------- refusals
def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        trb.plan_step(i, i, i[None].repeat(2, 1), i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        trb.release_pages(i, i, i[None].repeat(2, 1), i, i[:1], 16)
    with pytest.raises(ValueError, match="CUDA"):
        trb.append_kv(f[None], f[None], f[None, None], f[None, None], i.long())
    with pytest.raises(ValueError, match="CUDA"):
        trb.paged_attention(f[None], f[None, None], f[None, None], i[None], i, i)
    with pytest.raises(ValueError, match="CUDA"):
        trb.residual_norm(f, f, pre=f[0])
    with pytest.raises(ValueError, match="CUDA"):
        trb.sample_tokens(f, f, f[:, 0])


@gpu
def test_refusals():
    q, kp, vp, tables, lens, starts = attention_case([20, 30], [1, 1], 4, 2, 64, 16, torch.bfloat16)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    k = torch.zeros(2, 2, 64, device=DEV, dtype=torch.bfloat16)
    free, one = i32([5, 6]), i32([2])
    h = torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16)
    w = h[0].clone()
    lg, heat = torch.zeros(2, 9, device=DEV), torch.ones(2, device=DEV)
    bad = [
        lambda: trb.plan_step(lens.long(), lens, tables, free, one, 16, 2),
        lambda: trb.plan_step(lens, lens[:1], tables, free, one, 16, 2),
        lambda: trb.plan_step(lens, lens, tables[:1], free, one, 16, 2),
        lambda: trb.plan_step(lens, lens, tables.t().contiguous().t(), free, one, 16, 2),
        lambda: trb.plan_step(lens, lens, tables, free, free, 16, 2),
        lambda: trb.plan_step(lens, lens, tables, free, one, 0, 2),
        lambda: trb.plan_step(lens, lens, tables, free, one, 16, -1),
        lambda: trb.release_pages(lens, lens[:1], tables, free, one, 16),
        lambda: trb.append_kv(k, k[:1], kp, vp, slots),
        lambda: trb.append_kv(k.half(), k.half(), kp, vp, slots),
        lambda: trb.append_kv(k[:, :1], k[:, :1], kp, vp, slots),
        lambda: trb.append_kv(k, k, kp, vp[:1], slots),
        lambda: trb.append_kv(k, k, kp.transpose(1, 2), vp.transpose(1, 2), slots),
        lambda: trb.append_kv(k, k, kp, vp, slots.int()),
        lambda: trb.append_kv(k, k, kp, vp, slots[:1]),
        lambda: trb.paged_attention(q.half(), kp, vp, tables, lens, starts),
        lambda: trb.paged_attention(q[:, :3], kp, vp, tables, lens, starts),
        lambda: trb.paged_attention(q[..., :32], kp, vp, tables, lens, starts),
        lambda: trb.paged_attention(q, kp, vp, tables, lens, starts[:2]),
        lambda: trb.paged_attention(q, kp, vp, tables[:1], lens, starts),
        lambda: trb.paged_attention(q, kp, vp, tables, lens.long(), starts),
        lambda: trb.paged_attention(q, kp, vp, tables, lens, starts, scale=0.0),
        lambda: trb.paged_attention(q, kp, vp, tables, lens, starts, scale=math.inf),
        lambda: trb.residual_norm(h, h, pre=w[:5]),
        lambda: trb.residual_norm(h[:1], h, pre=w),
        lambda: trb.residual_norm(h.half(), h, pre=w),
        lambda: trb.residual_norm(None, h, pre=w, post=w),
        lambda: trb.residual_norm(None, h, pre=w, gate=w),
        lambda: trb.residual_norm(None, h),
        lambda: trb.residual_norm(h, h, pre=w.float()),
        lambda: trb.residual_norm(h, h, post_bias=w, pre=w),
        lambda: trb.residual_norm(h, h, pre=w, kind="batch"),
        lambda: trb.residual_norm(h, h, pre=w, eps=-1.0),
        lambda: trb.residual_norm(h, h, pre=w, eps=math.nan),
        lambda: trb.sample_tokens(lg, lg[:, :8], heat),
        lambda: trb.sample_tokens(lg, lg.half(), heat),
        lambda: trb.sample_tokens(lg.double(), lg, heat),
        lambda: trb.sample_tokens(lg, lg, heat[:1]),
        lambda: trb.sample_tokens(lg, lg, heat, top_k=heat),
        lambda: trb.sample_tokens(lg, lg, heat, top_p=lens),
        lambda: trb.sample_tokens(lg[:, :0], lg[:, :0], heat),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was accepted")
    unsupported = [
        lambda: trb.paged_attention(torch.zeros(1, 1, 264, device=DEV), torch.zeros(1, 1, 16, 264, device=DEV),
                                    torch.zeros(1, 1, 16, 264, device=DEV), i32([[0]]), i32([1]),
                                    i32([0, 1])),
        lambda: trb.paged_attention(torch.zeros(1, 1, 64, device=DEV), torch.zeros(1, 1, 24, 64, device=DEV),
                                    torch.zeros(1, 1, 24, 64, device=DEV), i32([[0]]), i32([1]),
                                    i32([0, 1])),
        lambda: trb.residual_norm(None, torch.zeros(1, 32776, device=DEV), pre=torch.ones(32776, device=DEV)),
        lambda: trb.plan_step(i32([0] * 16385), i32([0] * 16385), i32([[0]] * 16385), free, one, 16, 2),
    ]
    for call in unsupported:
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
