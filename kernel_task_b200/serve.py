"""The operators a decoder runs between its tensor-ring projections: the paged cache's step plan
and writes, attention over it, the norms around a block and sampling.

    step = plan_step(lens, new, tables, free, free_count, page_size, tokens)
    append_kv(k, v, k_pages, v_pages, step.slots)
    out = paged_attention(q, k_pages, v_pages, tables, step.lens, step.starts)
    h, x = residual_norm(o_proj.accumulate(out.flatten(1)), h, post=w0, pre=w1, gate=g)
    ids, logprobs = sample_tokens(logits, noise, temperature, top_k=k, top_p=p)

Each is one call of this library's CUDA kernels on the caller's current stream; none waits for
the GPU or reads anything back, so a step can be captured in a CUDA graph.  ValueError for wrong
shapes, types and devices, RuntimeError for what this build or the device cannot do.  CPU tensors
are refused; there is no fallback.  The reference has no counterpart: its decode chain leaves
attention, norms and sampling out (tools/qwen_model_chain.py:111-134).

The paged cache.  Keys and values live in two pools [pages, kv_heads, page_size, head_dim]; a
request's token at position p is in page ``tables[r, p // page_size]``, row p % page_size; its
slot is page * page_size + row.  Ids of free pages are a stack, ``free[:free_count]``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._native import binding


class StepPlan(NamedTuple):
    """What one step's tokens need; the tokens are numbered request by request.  The tensors of
    a plan share one allocation."""

    slots: torch.Tensor       # int64 [tokens], -1 where there is no token or its request is refused
    positions: torch.Tensor   # int32 [tokens], the token's position in its request, or -1
    starts: torch.Tensor      # int32 [requests + 1], first token of each request
    lens: torch.Tensor        # int32 [requests], tokens cached once the step's are appended
    granted: torch.Tensor     # int32 [requests], 0 where the request did not get its pages
    free_count: torch.Tensor  # int32 [1]


def plan_step(lens: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor,
              free_count: torch.Tensor, page_size: int, tokens: int, *,
              inplace: bool = False) -> StepPlan:
    """Block tables and slot maps of one step, built on the GPU from the requests' lengths.

    lens, new: int32 [requests], tokens cached and tokens brought (0 for an idle request);
    tables: int32 [requests, columns], the new pages' entries are written in place;
    free, free_count: the stack of free pages, int32 [pool] and int32 [1]; pages are taken in
    request order from its top, ``free`` itself stays; tokens: the size of the slot map, at
    least the sum of ``new`` (what is left over is padding).

    A request is refused, and keeps its length, when its pages would pass the table's columns,
    its tokens the slot map, or the pages needed up to and including it the free ones.
    ``inplace=True`` writes the new lengths and count into ``lens`` and ``free_count`` (a step
    captured in a CUDA graph); up to 16384 requests.
    """
    return StepPlan._make(binding().plan_step(lens, new, tables, free, free_count, page_size,
                                              tokens, inplace))


def release_pages(lens: torch.Tensor, finished: torch.Tensor, tables: torch.Tensor,
                  free: torch.Tensor, free_count: torch.Tensor, page_size: int) -> None:
    """Give the pages of the requests with ``finished`` (int32 [requests]) back to the stack, in
    place: their table entries become -1, their lens 0, and free_count grows."""
    binding().release_pages(lens, finished, tables, free, free_count, page_size)


def append_kv(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              slots: torch.Tensor) -> None:
    """Write k, v [tokens, kv_heads, head_dim] (any strides; the pools' dtype, or float32 rounded
    to it) to their slots (int64 [tokens], all different).  Negative slots and slots past the
    pools are skipped."""
    binding().append_kv(k, v, k_pages, v_pages, slots)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    tables: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor, *,
                    scale: float | None = None, return_lse: bool = False):
    """Causal attention of each request's last tokens over its paged cache.

    q: [tokens, heads, head_dim], request r's tokens in rows starts[r]:starts[r + 1]; they are
    the last of its lens[r] cached tokens, so token i sees positions up to
    lens[r] - n_r + i.  Query head h reads kv head h // (heads // kv_heads).  Cache rows at and
    past lens[r] are never used; a token that sees none gives zeros.  ``scale`` is
    head_dim ** -0.5 by default.  Returns out [tokens, heads, head_dim] in q's dtype, and with
    ``return_lse`` also the fp32 log of the sum of exponentials [tokens, heads] (-inf for none).

    float16 and bfloat16 with head_dim 64 or 128 run on tensor cores, other multiples of 8 up to
    256 and float32 on a general kernel.  The page size is a power of two up to 1024.
    Values of a request's own tokens have to be finite: a later token's infinity or NaN may reach
    earlier tokens of the same call; what lies past the length may be anything.
    """
    out, lse = binding().paged_attention(q, k_pages, v_pages, tables, lens, starts, scale,
                                         return_lse)
    return (out, lse) if return_lse else out


def attention_status(device: torch.device | str | int | None = None, *, reset: bool = True) -> int:
    """0, or ``abi.TR_ERR_TIMEOUT`` when a bounded wait inside a ``paged_attention`` on the current
    stream of ``device`` gave up; waits for the stream.

    What such a call did not finish is NaN, and all that later calls on the stream give, until this
    function has found the timeout (``reset``: the next call starts from a new workspace).  A call
    captured in a CUDA graph has a workspace of its own, which every replay zeroes: a timeout shows
    in the NaN of that replay alone.  With ``TRR_CHECK_STATUS=1`` in the environment every call
    outside a capture asks by itself, and raises RuntimeError."""
    d = torch.device("cuda" if device is None else device)
    return binding().attention_status(torch.cuda.current_device() if d.index is None else d.index,
                                      reset)


def set_attention_wait_limit(polls: int) -> None:
    """Polls that a wait inside ``paged_attention`` makes before it gives up, in all calls from now on
    (0: the built-in limit, about a second).  For tests of the timeout path."""
    binding().set_attention_wait_limit(polls)


def residual_norm(y: torch.Tensor | None, h: torch.Tensor, *, post: torch.Tensor | None = None,
                  pre: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, pre_bias: torch.Tensor | None = None,
                  kind: str = "rms", eps: float = 1e-6, residual_scale: float = 1.0,
                  branch_scale: float = 1.0):
    """The norms after and before a block, with the block's gate and the scaled residual add:

        h' = residual_scale * h + branch_scale * gate * norm(y; post)
        x' = norm(h'; pre)

    y [tokens, width] is the block's output, float32 (``op.accumulate``) or h's dtype; None norms
    h alone.  post, pre (and the biases, for kind="layer" or "rms" alike): [width]; without
    ``post`` y is added as it is, without ``pre`` there is no x'.  gate: None, [width] or
    [tokens, width].  kind: "rms" or "layer" (mean removed).  All in h's dtype but y.  The sums
    are fp32, x' is normed from the unrounded h', and each output is rounded once.
    Returns (h', x'), with h itself where y is None and None where pre is.  Widths to 32768.
    """
    return binding().residual_norm(y, h, post, pre, gate, post_bias, pre_bias, kind, eps,
                                   residual_scale, branch_scale)


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor, temperature: torch.Tensor, *,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None):
    """The next token of every row of logits [rows, vocab] from given random numbers.

    noise: float32 [rows, vocab] ~ Exp(1) (``torch.Tensor.exponential_``); temperature, top_p,
    min_p: float32 [rows]; top_k: int32 [rows].  Of the softmax of t = logits / temperature are
    kept the top_k greatest (0: all), of these the shortest run in falling order whose mass
    reaches top_p of theirs (1: all), of these the ones of at least min_p times the greatest.
    The token is the kept one with the greatest t - log(noise), which draws it with its
    probability among the kept, or at temperature 0 the one with the greatest logit.  Ranks and
    cuts are those of the logits, also where t no longer tells them apart: an infinite temperature
    draws evenly among what the limits keep.  Ties of logits go to the lower index everywhere.  The
    greatest token is always kept; NaN logits count as -inf; a row of nothing but -inf gives token
    -1.  The same call gives the same bits; a row's masses are summed in an order that depends on
    the number of rows too, so a cut or a logprob may differ in its last bits between batches.

    Returns (tokens int64 [rows], logprobs float32 [rows]): the log of the token's probability
    in the softmax of t over the whole row.
    """
    return binding().sample_tokens(logits, noise, temperature, top_k, top_p, min_p)
