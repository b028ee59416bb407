"""Numpy float64 restatements of the serving operators (kernel_task_b200/serve.py), written from
their definitions, one request or row at a time.  Test infrastructure only."""
from __future__ import annotations

import numpy as np


def plan_step(lens, new, tables, free, free_count, page_size, tokens):
    """Serial step plan: (slots, positions, starts, lens, granted, free_count, tables)."""
    R, columns = len(lens), tables.shape[1]
    tables = tables.copy()
    slots = np.full(tokens, -1, np.int64)
    positions = np.full(tokens, -1, np.int32)
    starts = np.zeros(R + 1, np.int32)
    out_lens, granted = np.array(lens, np.int32), np.zeros(R, np.int32)
    asked, taken = 0, 0  # pages asked for by the requests that fit, pages given
    for r in range(R):
        n, held_tokens = max(int(new[r]), 0), max(int(lens[r]), 0)
        starts[r + 1] = starts[r] + n
        held, wants = -(-held_tokens // page_size), -(-(held_tokens + n) // page_size)
        if wants > columns or starts[r + 1] > tokens:
            continue
        need = wants - held
        asked += need
        if need > 0 and asked > free_count:
            continue
        granted[r] = 1
        for c in range(held, wants):
            tables[r, c] = free[free_count - 1 - (asked - need) - (c - held)]
        taken = asked if need > 0 else taken
        for i in range(n):
            p = held_tokens + i
            slots[starts[r] + i] = int(tables[r, p // page_size]) * page_size + p % page_size
            positions[starts[r] + i] = p
        out_lens[r] = held_tokens + n
    return slots, positions, starts, out_lens, granted, free_count - taken, tables


def gather(pages, table, length):
    """Rows 0 .. length - 1 of one request: [length, kv_heads, head_dim]; bad page ids give zeros."""
    P, H, size, D = pages.shape
    out = np.zeros((length, H, D))
    for j in range(length):
        page = int(table[j // size])
        if 0 <= page < P:
            out[j] = pages[page, :, j % size]
    return out


def paged_attention(q, k_pages, v_pages, tables, lens, starts, scale):
    """(out, lse, spread): spread = sum_j p_j |v_j|, what rounding errors of p scale with."""
    T, H, D = q.shape
    G = k_pages.shape[1]
    out, spread = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse = np.full((T, H), -np.inf)
    for r in range(len(lens)):
        a, b = int(starts[r]), int(starts[r + 1])
        length = min(int(lens[r]), tables.shape[1] * k_pages.shape[2])
        if length <= 0 or b <= a:
            continue
        K, V = gather(k_pages, tables[r], length), gather(v_pages, tables[r], length)
        for i in range(b - a):
            n = min(length, int(lens[r]) - (b - a) + i + 1)
            if n <= 0:
                continue
            for h in range(H):
                g = h // (H // G)
                s = scale * (K[:n, g] @ q[a + i, h])
                m = s.max()
                e = np.exp(s - m)
                out[a + i, h] = e @ V[:n, g] / e.sum()
                spread[a + i, h] = e @ np.abs(V[:n, g]) / e.sum()
                lse[a + i, h] = m + np.log(e.sum())
    return out, lse, spread


def residual_norm(y, h, post=None, pre=None, gate=None, post_bias=None, pre_bias=None, kind="rms",
                  eps=1e-6, residual_scale=1.0, branch_scale=1.0):
    def norm(v, weight, bias):
        if kind == "layer":
            v = v - v.mean(-1, keepdims=True)
        v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * weight
        return v if bias is None else v + bias

    if y is not None:
        branch = y if post is None else norm(y, post, post_bias)
        branch = branch if gate is None else branch * gate
        h = residual_scale * h + branch_scale * branch
    return h, None if pre is None else norm(h, pre, pre_bias)


def sample(logits, noise, temperature, top_k=0, top_p=1.0, min_p=0.0, margin=0.0):
    """One row: (token, logprob, clear); clear is False when a decision was nearer than `margin`."""
    t = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    if temperature > 0:
        t = t / temperature
    top = t.max()
    if top == -np.inf:
        return -1, -np.inf, True
    w = np.where(t == top, 1.0, np.exp(np.where(t == top, 0.0, t - top)))
    logprob = np.where(t == top, 0.0, t - top) - np.log(w.sum())
    if not temperature > 0:
        token = int(np.flatnonzero(t == top)[0])
        return token, logprob[token], True
    clear = True
    kept = np.argsort(-t, kind="stable")
    if 0 < top_k < len(kept):
        kept = kept[:top_k]
    if top_p < 1:
        before = np.cumsum(w[kept]) - w[kept]
        target = top_p * w[kept].sum()
        clear &= not np.any(np.abs(before[1:] - target) < margin * w[kept].sum())
        within = before < target
        within[0] = True
        kept = kept[within]
    floor = min(min_p, 1.0)
    clear &= not np.any(np.abs(w[kept] - floor)[w[kept] < 1] < margin * floor)
    kept = kept[(w[kept] >= floor) & (t[kept] > -np.inf)]
    key = t[kept] - np.log(noise[kept].astype(np.float64))
    best = key.max()
    second = np.sort(key)[-2] if len(key) > 1 else -np.inf
    clear &= bool(best - second > margin) or margin == 0
    token = int(kept[key == best].min())
    return token, logprob[token], bool(clear)
