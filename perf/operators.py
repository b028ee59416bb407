"""The serving operators that stand around the tensor-ring projections of a decoder, as cases to
measure: sizes, inputs, a plain form in elementary torch operations, and the same results in 64
bits.

  plan     block tables and slot maps of one step from the requests' lengths
  append   new keys and values written into the paged cache
  attend   attention of each request's new tokens over its paged cache
  norm     norms after and before a block, with the gate and the scaled residual add between
  sample   the next token from logits with temperature, top-k, top-p and min-p

A decoder step runs them in this order; the projections between them are the tensor-ring
operators.  Head layouts (32 query heads over 8 of 128) and widths (4096, 2880) are those of the
projections this repository benchmarks.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a busy server: every request brings one token, few need a page
        dict(name="plan_decode", op="plan", requests=256, context=8192, new=1, page=16,
             short=False),
        # prompts admitted together: 65536 tokens in ragged pieces, the pool too small for all
        dict(name="plan_prompts", op="plan", requests=500, context=4096, new=256, page=64,
             short=True),
        # the cache write of one decode step of 128 requests, a slice of the fused projection
        dict(name="append_decode", op="append", tokens=128, kv_heads=8, head_dim=128, page=16,
             dtype="bf16", source="bf16"),
        # a prompt's cache write from fp32 projection outputs
        dict(name="append_prompt", op="append", tokens=32771, kv_heads=8, head_dim=128, page=32,
             dtype="bf16", source="fp32"),
        # a single user's next token, a short odd context: latency
        dict(name="attend_one", op="attend", requests=1, context=777, new=1, mixed=0.0, heads=32,
             kv_heads=8, head_dim=128, page=16, dtype="bf16"),
        # a batch of decoding requests with ragged contexts, one token each
        dict(name="attend_batch", op="attend", requests=61, context=16384, new=1, mixed=0.0,
             heads=32, kv_heads=8, head_dim=128, page=16, dtype="bf16"),
        # a mixed step: chunks of prompts next to requests that decode
        dict(name="attend_mixed", op="attend", requests=12, context=8192, new=512, mixed=0.5,
             heads=32, kv_heads=8, head_dim=128, page=64, dtype="bf16"),
        # whole prompts with nothing cached before them
        dict(name="attend_prompts", op="attend", requests=3, context=0, new=4099, mixed=0.0,
             heads=28, kv_heads=4, head_dim=64, page=32, dtype="fp16"),
        # between two blocks of a decode step, from the fp32 output of a projection
        dict(name="norm_decode", op="norm", tokens=1, width=4096, kind="rms", gate="channel",
             dtype="bf16", source="fp32"),
        # the same over a prefill of an uneven length, gated per token, mean removed
        dict(name="norm_prefill", op="norm", tokens=16391, width=2880, kind="layer", gate="token",
             dtype="fp16", source="fp16"),
        # one user's next token from fp32 logits of an odd vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=50021, dtype="fp32"),
        # a server's step: every row with settings of its own
        dict(name="sample_batch", op="sample", rows=256, vocab=131072, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "norm", "sample"])
    half = rng.choice(["bf16", "fp16"])
    if op == "plan":
        requests = _log(rng, 1, 1000)
        return dict(op=op, requests=requests, context=_log(rng, 16, 16384),
                    new=_log(rng, 1, max(1, 65536 // requests)), page=rng.choice([16, 32, 64, 128]),
                    short=rng.random() < 0.3)
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 32768), kv_heads=rng.choice([1, 2, 4, 5, 8]),
                    head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), dtype=half,
                    source=rng.choice([half, "fp32"]))
    if op == "attend":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        heads = heads if heads <= 32 else kv_heads * 4
        shape = dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128]),
                     page=rng.choice([16, 32, 64, 128]), dtype=half)
        if rng.random() < 0.5:
            requests = _log(rng, 1, 64)
            return dict(op=op, requests=requests, context=_log(rng, 1, min(65536, 800000 // requests)),
                        new=1, mixed=0.0, **shape)
        requests = rng.randint(1, 8)
        new = _log(rng, 2, 3500 // requests)
        return dict(op=op, requests=requests, context=rng.choice([0, _log(rng, 1, 7000)]), new=new,
                    mixed=rng.choice([0.0, 0.5]), **shape)
    if op == "norm":
        width = rng.choice([1920, 2880, 4096, 14336, _log(rng, 33, 8192)])
        return dict(op=op, tokens=_log(rng, 1, max(1, 47000000 // width)), width=width,
                    kind=rng.choice(["rms", "layer"]), gate=rng.choice(["none", "channel", "token"]),
                    dtype=half, source=rng.choice([half, "fp32"]))
    return dict(op=op, rows=_log(rng, 1, 200), vocab=_log(rng, 1000, 131072),
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


# ------------------------------------------------------------------------- lengths of a case
def _lengths(case):
    """Tokens each request holds before the step and brings with it: of the case alone."""
    r = random.Random("%(requests)d/%(context)d/%(new)d/%(page)d" % case)
    n, context, new = case["requests"], case["context"], case["new"]
    mixed = case.get("mixed", 0.0)
    held = [0 if context == 0 else context if i == 0 else max(1, int(context * r.random() ** 1.5))
            for i in range(n)]
    brings = [new if new == 1 or i == 0 else 1 if r.random() < mixed else r.randint(max(1, new // 4), new)
              for i in range(n)]
    return held, brings


def _pages(length, page):
    return -(-length // page)


def _pool(counts, spare, columns, gen):
    """A table of pages in random order, `counts` per row, and the pages left over."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    have = torch.tensor(counts, device="cuda")
    column = torch.arange(columns, device="cuda")[None, :]
    at = (have.cumsum(0) - have)[:, None] + column
    table = torch.where(column < have[:, None], order[at.clamp(max=total - 1)],
                        torch.full_like(at, -1, dtype=torch.int32))
    return table.contiguous(), order[sum(counts):].contiguous(), total


# --------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    if op == "plan":
        held, brings = _lengths(case)
        page = case["page"]
        # a server has idle requests too: every seventh brings nothing this step
        brings = [0 if i % 7 == 3 else b for i, b in enumerate(brings)]
        need = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(held, brings))
        columns = max(_pages(a + b, page) for a, b in zip(held, brings)) + 3
        spare = need * 2 // 3 if case["short"] else need + 17
        table, free, _ = _pool([_pages(a, page) for a in held], max(1, spare), columns, gen)
        tokens = sum(brings) + 5
        return dict(case=case, lens=torch.tensor(held, dtype=torch.int32, device="cuda"),
                    new=torch.tensor(brings, dtype=torch.int32, device="cuda"), tables=table,
                    free=free, free_count=torch.tensor([free.numel()], dtype=torch.int32, device="cuda"),
                    tokens=tokens)
    if op == "append":
        T, H, D, page = case["tokens"], case["kv_heads"], case["head_dim"], case["page"]
        # keys and values are slices of one projection's output, so their rows are strided
        both = normal(T, 2 * H * D, dtype=_TYPES[case["source"]])
        k, v = both[:, :H * D].unflatten(1, (H, D)), both[:, H * D:].unflatten(1, (H, D))
        pages = _pages(T, page) + 9
        table, _, _ = _pool([_pages(T, page)], 9, _pages(T, page), gen)
        at = torch.arange(T, device="cuda")
        slots = table[0].long()[at // page] * page + at % page
        if T > 3:
            slots[T - 2:] = -1  # a step's padding
        shape = (pages, H, page, D)
        return dict(case=case, k=k, v=v, slots=slots, k_pages=normal(*shape, dtype=_TYPES[case["dtype"]]),
                    v_pages=normal(*shape, dtype=_TYPES[case["dtype"]]))
    if op == "attend":
        held, brings = _lengths(case)
        page, D, H = case["page"], case["head_dim"], case["heads"]
        lens = [a + b for a, b in zip(held, brings)]
        columns = max(_pages(n, page) for n in lens) + 2
        table, _, total = _pool([_pages(n, page) for n in lens], 3, columns, gen)
        kind = _TYPES[case["dtype"]]
        shape = (total, case["kv_heads"], page, D)
        # queries are a slice of the fused projection; keys have a shared part, as trained ones do
        both = normal(sum(brings), (H + 2 * case["kv_heads"]) * D, dtype=kind)
        q = both[:, :H * D].unflatten(1, (H, D))
        k_pages = normal(*shape, dtype=kind).add_(normal(1, case["kv_heads"], 1, D, dtype=kind))
        n = torch.tensor(brings, dtype=torch.int32, device="cuda")
        starts = torch.zeros(len(brings) + 1, dtype=torch.int32, device="cuda")
        starts[1:] = n.cumsum(0)
        return dict(case=case, q=q, k_pages=k_pages, v_pages=normal(*shape, dtype=kind), tables=table,
                    lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), starts=starts,
                    longest=max(lens), most=max(brings))
    if op == "norm":
        T, W, kind = case["tokens"], case["width"], _TYPES[case["dtype"]]
        gate = {"none": None, "channel": lambda: normal(W, dtype=kind, scale=0.5),
                "token": lambda: normal(T, W, dtype=kind, scale=0.5)}[case["gate"]]
        layer = case["kind"] == "layer"
        return dict(case=case, y=normal(T, W, dtype=_TYPES[case["source"]]).mul_(3.0).add_(0.25),
                    h=normal(T, W, dtype=kind).mul_(2.0), gate=gate and gate(),
                    post=normal(W, dtype=kind, scale=0.1).add_(1.0),
                    pre=normal(W, dtype=kind, scale=0.1).add_(1.0),
                    post_bias=normal(W, dtype=kind, scale=0.1) if layer else None,
                    pre_bias=normal(W, dtype=kind, scale=0.1) if layer else None)
    R, V = case["rows"], case["vocab"]
    # a body of unlikely tokens and a few likely ones; some rows under a grammar's mask
    logits = normal(R, V, scale=2.0)
    likely = torch.randint(V, (R, 24), generator=gen, device="cuda")
    logits.scatter_add_(1, likely, normal(R, 24).abs_().mul_(5.0))
    row = torch.arange(R, device="cuda")[:, None]
    banned = (torch.rand(R, V, generator=gen, device="cuda") < 0.3) & (row % 4 == 3)
    logits.masked_fill_(banned, -math.inf)

    def pick(values, dtype):
        at = torch.randint(len(values), (R,), generator=gen, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    noise = torch.empty(R, V, device="cuda").exponential_(generator=gen)
    return dict(case=case, logits=logits.to(_TYPES[case["dtype"]]), noise=noise,
                temperature=pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32),
                top_k=pick([0, 1, 20, 50, 400], torch.int32),
                top_p=pick([1.0, 0.95, 0.9, 0.5], torch.float32),
                min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))


# ------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _RUN[case["op"]](state)
    return _PLAIN[case["op"]](state)


def _run_plan(s):
    from kernel_task_b200 import plan_step
    step = plan_step(s["lens"], s["new"], s["tables"], s["free"], s["free_count"],
                     s["case"]["page"], s["tokens"])
    return [step.slots, step.positions, step.starts, step.lens, step.granted, step.free_count,
            s["tables"]]


def _run_append(s):
    from kernel_task_b200 import append_kv
    append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
    return [s["k_pages"], s["v_pages"]]


def _run_attend(s):
    from kernel_task_b200 import paged_attention
    return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["starts"],
                           return_lse=True)


def _run_norm(s):
    from kernel_task_b200 import residual_norm
    return residual_norm(s["y"], s["h"], post=s["post"], pre=s["pre"], gate=s["gate"],
                         post_bias=s["post_bias"], pre_bias=s["pre_bias"], kind=s["case"]["kind"],
                         eps=1e-5, residual_scale=1.0, branch_scale=0.5)


def _run_sample(s):
    from kernel_task_b200 import sample_tokens
    return sample_tokens(s["logits"], s["noise"], s["temperature"], top_k=s["top_k"],
                         top_p=s["top_p"], min_p=s["min_p"])


_RUN = {"plan": _run_plan, "append": _run_append, "attend": _run_attend, "norm": _run_norm,
        "sample": _run_sample}


# ------------------------------------------------------------------------------ plain forms
def _plain_plan(s):
    lens, new, tables, page, T = s["lens"], s["new"], s["tables"], s["case"]["page"], s["tokens"]
    columns = tables.shape[1]
    starts = torch.zeros(lens.numel() + 1, dtype=torch.int32, device=lens.device)
    starts[1:] = new.cumsum(0)
    held = (lens + page - 1) // page
    wants = (lens + new + page - 1) // page
    fits = (wants <= columns) & (starts[1:] <= T)
    need = torch.where(fits, wants - held, 0)
    through = need.cumsum(0)
    granted = fits & ((need == 0) | (through <= s["free_count"]))
    # request r takes the pages below the top of the free stack, after those of earlier requests
    column = torch.arange(columns, device=lens.device)[None, :]
    takes = granted[:, None] & (column >= held[:, None]) & (column < wants[:, None])
    at = s["free_count"] - 1 - ((through - need)[:, None] + column - held[:, None])
    tables.copy_(torch.where(takes, s["free"][at.clamp(0, s["free"].numel() - 1).long()], tables))
    token = torch.arange(T, device=lens.device, dtype=torch.int32)
    owner = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    inside = owner < lens.numel()
    owner = owner.clamp(max=lens.numel() - 1)
    inside &= granted[owner]
    position = lens[owner] + token - starts[:-1][owner]
    block = (position // page).clamp(max=columns - 1).long()
    slot = tables[owner, block].long() * page + position % page
    used = torch.where(granted, need, 0).sum(dtype=torch.int32)
    return [torch.where(inside, slot, -1), torch.where(inside, position, -1), starts,
            torch.where(granted, lens + new, lens), granted.to(torch.int32), s["free_count"] - used,
            tables]


def _plain_append(s):
    k_pages, v_pages, page = s["k_pages"], s["v_pages"], s["case"]["page"]
    kept = torch.nonzero(s["slots"] >= 0)[:, 0] if s["slots"].numel() <= 3 else slice(0, -2)
    slot = s["slots"][kept]
    k_pages[slot // page, :, slot % page] = s["k"][kept].to(k_pages.dtype)
    v_pages[slot // page, :, slot % page] = s["v"][kept].to(v_pages.dtype)
    return [k_pages, v_pages]


def _plain_attend(s):
    case, q, tables, lens, starts = s["case"], s["q"], s["tables"], s["lens"], s["starts"]
    G, D, page, H = case["kv_heads"], case["head_dim"], case["page"], case["heads"]
    R, L, N = lens.numel(), s["longest"], s["most"]
    blocks = _pages(L, page)
    at = tables[:, :blocks].clamp(min=0).long()

    def laid_out(pages):  # [R, G, blocks * page, D]
        return pages[at].transpose(1, 2).reshape(R, G, blocks * page, D)[:, :, :L].float()

    new = starts[1:] - starts[:-1]
    i = torch.arange(N, device=q.device)
    j = torch.arange(L, device=q.device)
    row = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1).long()
    qs = q[row].float().reshape(R, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(R, G, -1, D)
    scores = (qs @ laid_out(s["k_pages"]).transpose(2, 3)).mul_(D ** -0.5)
    scores = scores.view(R, G, H // G, N, L)
    seen = j <= (lens - new)[:, None, None] + i[:, None]
    seen = seen & (i[:, None] < new[:, None, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = scores.sum(-1, keepdim=True)
    values = laid_out(s["v_pages"]) * (j[:, None] < lens[:, None, None, None])
    out = (scores.view(R, G, -1, L) @ values).view(R, G, H // G, N, D)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (most + torch.log(total)).squeeze(-1)
    # back to one row per token
    token = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
    owner = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    inner = (token - starts[:-1][owner]).long()
    out = out.permute(0, 3, 1, 2, 4)[owner, inner].reshape(-1, H, D).to(q.dtype)
    return out, lse.permute(0, 3, 1, 2)[owner, inner].reshape(-1, H)


def _plain_norm(s):
    layer = s["case"]["kind"] == "layer"

    def norm(x, weight, bias):
        x = x - x.mean(-1, keepdim=True) if layer else x
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight.float()
        return x if bias is None else x + bias.float()

    branch = norm(s["y"].float(), s["post"], s["post_bias"])
    branch = branch if s["gate"] is None else branch * s["gate"].float()
    h = s["h"].float() + 0.5 * branch
    x = norm(h, s["pre"], s["pre_bias"])
    return h.to(s["h"].dtype), x.to(s["h"].dtype)


def _plain_sample(s):
    V = s["logits"].shape[1]
    heat = s["temperature"][:, None]
    t = s["logits"].float() / torch.where(heat > 0, heat, 1.0)
    top = t.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    w = torch.where(t == base, 1.0, torch.exp(t - base))
    total = w.sum(-1, keepdim=True)
    t, order = torch.sort(t, dim=-1, descending=True, stable=True)
    w = w.gather(1, order)
    k = s["top_k"][:, None]
    keep = torch.arange(V, device=t.device) < torch.where(k > 0, k, V)
    w = w * keep
    before = w.cumsum(-1) - w
    p = s["top_p"][:, None]
    keep &= (p >= 1) | (before < p * w.sum(-1, keepdim=True))
    keep &= (w >= s["min_p"][:, None]) & (t > -math.inf)
    key = torch.where(heat > 0, t - torch.log(s["noise"].gather(1, order)), t)
    key = torch.where(keep, key, -math.inf)
    best = key.amax(-1, keepdim=True)
    token = torch.where((key == best) & keep, order, V).amin(-1, keepdim=True)
    none = token == V
    token = torch.where(none, 0, token)
    chosen = s["logits"].gather(1, token).float() / torch.where(heat > 0, heat, 1.0)
    gap = torch.where(chosen == base, 0.0, chosen - base)
    logprob = torch.where(none, -math.inf, gap - torch.log(total))
    return torch.where(none, -1, token)[:, 0], logprob[:, 0]


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
          "norm": _plain_norm, "sample": _plain_sample}


# ---------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "plan":
        held, brings = _lengths(case)
        page = case["page"]
        n = case["requests"]
        brings = [0 if i % 7 == 3 else b for i, b in enumerate(brings)]
        need = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(held, brings))
        # lengths in and out, starts, grants; a page moved from the stack to a table; per token
        # a slot, a position and the table entry of the blocks it touches
        return {"bytes": n * 20 + need * 8 + sum(brings) * 12 + sum(_pages(b, page) for b in brings) * 4,
                "flops": 0}
    if op == "append":
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": n * (_BYTES[case["dtype"]] + _BYTES[case["source"]]) + case["tokens"] * 8,
                "flops": 0}
    if op == "attend":
        held, brings = _lengths(case)
        H, G, D = case["heads"], case["kv_heads"], case["head_dim"]
        pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(held, brings))
        cached = sum(a + b for a, b in zip(held, brings))
        return {"bytes": 2 * cached * G * D * 2 + sum(brings) * H * (D * 4 + 4)
                + 4 * sum(_pages(a + b, case["page"]) for a, b in zip(held, brings)),
                "flops": 4 * pairs * H * D}
    if op == "norm":
        n, b = case["tokens"] * case["width"], _BYTES[case["dtype"]]
        gate = {"none": 0, "channel": case["width"] * b, "token": n * b}[case["gate"]]
        params = (4 if case["kind"] == "layer" else 2) * case["width"] * b
        return {"bytes": n * (_BYTES[case["source"]] + 3 * b) + gate + params, "flops": 12 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (_BYTES[case["dtype"]] + 4) + case["rows"] * 28, "flops": 4 * n}


# ------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend,
            "norm": _exact_norm, "sample": _exact_sample}[case["op"]](s)


def _exact_plan(s):
    return None  # whole numbers only


def _exact_append(s):
    page = s["case"]["page"]
    slots = s["slots"].cpu().numpy()
    kept = np.flatnonzero(slots >= 0)
    k_pages, v_pages = s["k_pages"].double().cpu().numpy(), s["v_pages"].double().cpu().numpy()
    k_pages[slots[kept] // page, :, slots[kept] % page] = s["k"].double().cpu().numpy()[kept]
    v_pages[slots[kept] // page, :, slots[kept] % page] = s["v"].double().cpu().numpy()[kept]
    return [k_pages, v_pages]


def _exact_rows(s, r):
    """One request's outputs and log-sums, its keys and values read page by page."""
    case = s["case"]
    page, G, H, D = case["page"], case["kv_heads"], case["heads"], case["head_dim"]
    first, last, length = int(s["starts"][r]), int(s["starts"][r + 1]), int(s["lens"][r])
    ids = s["tables"][r, :_pages(length, page)].long()
    keys = torch.cat(list(s["k_pages"][ids].double()), dim=1)[:, :length]
    values = torch.cat(list(s["v_pages"][ids].double()), dim=1)[:, :length]
    last_seen = torch.arange(length - (last - first), length, device=keys.device)
    hidden = torch.arange(length, device=keys.device)[None, :] > last_seen[:, None]

    def head(h):
        a = torch.einsum("nd,ld->nl", s["q"][first:last, h].double(), keys[h // (H // G)])
        a = (a / math.sqrt(D)).masked_fill(hidden, -math.inf)
        return torch.softmax(a, -1) @ values[h // (H // G)], torch.logsumexp(a, -1)

    got = [head(h) for h in range(H)]
    return torch.stack([o for o, _ in got], 1), torch.stack([e for _, e in got], 1)


def _exact_attend(s):
    rows = [_exact_rows(s, r) for r in range(s["lens"].numel())]
    return torch.cat([o for o, _ in rows]), torch.cat([e for _, e in rows])


def _exact_norm(s):
    f = lambda x: None if x is None else x.double().cpu().numpy()  # noqa: E731

    def norm(x, weight, bias):
        if s["case"]["kind"] == "layer":
            x = (x - x.mean(1)[:, None]) / np.sqrt(x.var(1)[:, None] + 1e-5)
            return x * weight + bias
        return x / np.sqrt((x * x).mean(1)[:, None] + 1e-5) * weight

    g = f(s["gate"])
    h = f(s["h"]) + 0.5 * (1.0 if g is None else g) * norm(f(s["y"]), f(s["post"]), f(s["post_bias"]))
    return h, norm(h, f(s["pre"]), f(s["pre_bias"]))


def _exact_sample(s):
    heat = s["temperature"].double().cpu().numpy()
    logits = s["logits"].double().cpu().numpy()
    noise = s["noise"].double().cpu().numpy()
    k, p, least = (s[n].cpu().numpy().astype(np.float64) for n in ("top_k", "top_p", "min_p"))

    def one(r):
        t = logits[r] / (heat[r] if heat[r] > 0 else 1.0)
        logprobs = t - t.max() - np.log(np.exp(t - t.max()).sum())
        order = np.argsort(-t, kind="stable")[:int(k[r]) if k[r] > 0 else t.size]
        mass = np.exp(t[order] - t.max())
        if p[r] < 1:
            before = np.concatenate([[0.0], mass.cumsum()[:-1]])
            order = order[before < p[r] * mass.sum()]
            mass = mass[:order.size]
        order = order[(mass >= least[r]) & np.isfinite(t[order])]
        key = t[order] - np.log(noise[r, order]) if heat[r] > 0 else t[order]
        token = order[key == key.max()].min()
        return token, logprobs[token]

    got = [one(r) for r in range(heat.size)]
    return np.array([g[0] for g in got], np.int64), np.array([g[1] for g in got])
