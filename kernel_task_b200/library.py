"""torch.library registration of the operator, so that prepared operators compose with
torch.compile, CUDA graphs and other custom-op machinery:

    handle = kernel_task_b200.library.register(fn, spec)     # fn from prepare_optimized
    y = torch.ops.trring.forward(x, handle)                  # same as fn(x)
    h = torch.ops.trring.forward_add(x, h0, handle)          # fn.forward_add(x, h0)
    a = torch.ops.trring.forward_silu_mul(x, g, handle)      # fn.forward_silu_mul(x, g)
    g = torch.ops.trring.accumulate(x, handle)               # fn.accumulate(x), fp32
    torch.ops.trring.consume_silu_mul(g, u), torch.ops.trring.consume_add(h, y)

and the serving operators (serve.py), with positional arguments:

    slots, positions, starts, lens, granted, free_count = torch.ops.trring.plan_step(
        lens, new, tables, free, free_count, page_size, tokens)
    torch.ops.trring.append_kv(k, v, k_pages, v_pages, slots)
    out, lse = torch.ops.trring.paged_attention(q, k_pages, v_pages, tables, lens, starts, scale)
    h, x = torch.ops.trring.residual_norm(y, h, post, pre, gate, post_bias, pre_bias, kind, eps,
                                          residual_scale, branch_scale)
    ids, logprobs = torch.ops.trring.sample_tokens(logits, noise, temperature, top_k, top_p, min_p)

A prepared operator is a C++ object, which a custom op cannot take as an argument, so operators
are registered in a process-local table and the op takes the integer handle.  Each op has a
fake (meta) implementation giving the output shape and dtype without running a kernel.
"""
from __future__ import annotations

import itertools
import threading
from typing import Optional

import torch

from . import serve as _serve
from ._native import binding
from .ring import consume_add as _consume_add
from .ring import consume_silu_mul as _consume_silu_mul
from .spec import TRSpec

_lock = threading.Lock()
_ids = itertools.count(1)
_table: dict[int, tuple[object, int, int]] = {}  # handle -> (operator, in_features, out_features)


def register(op, spec: TRSpec) -> int:
    """Make `op` (a prepared operator for `spec`) callable through torch.ops.trring.*."""
    with _lock:
        handle = next(_ids)
        _table[handle] = (op, spec.in_features, spec.out_features)
    return handle


def unregister(handle: int) -> None:
    with _lock:
        _table.pop(handle, None)


def _entry(handle: int, x: torch.Tensor):
    try:
        op, d_in, d_out = _table[handle]
    except KeyError:
        raise ValueError(f"no operator registered under handle {handle}") from None
    if x.dim() != 2 or x.shape[1] != d_in:
        raise ValueError(f"Expected x with shape [tokens, {d_in}]")
    return op, d_out


@torch.library.custom_op("trring::forward", mutates_args=())
def forward(x: torch.Tensor, handle: int) -> torch.Tensor:
    op, _ = _entry(handle, x)
    return op(x)


@forward.register_fake
def _(x, handle):
    _, d_out = _entry(handle, x)
    return x.new_empty((x.shape[0], d_out))


@torch.library.custom_op("trring::accumulate", mutates_args=())
def accumulate(x: torch.Tensor, handle: int) -> torch.Tensor:
    op, _ = _entry(handle, x)
    return op.accumulate(x)


@accumulate.register_fake
def _(x, handle):
    _, d_out = _entry(handle, x)
    return x.new_empty((x.shape[0], d_out), dtype=torch.float32)


@torch.library.custom_op("trring::forward_add", mutates_args=())
def forward_add(x: torch.Tensor, h: torch.Tensor, handle: int) -> torch.Tensor:
    op, _ = _entry(handle, x)
    return op.forward_add(x, h)


@forward_add.register_fake
def _(x, h, handle):
    _, d_out = _entry(handle, x)
    return x.new_empty((x.shape[0], d_out))


@torch.library.custom_op("trring::forward_silu_mul", mutates_args=())
def forward_silu_mul(x: torch.Tensor, g: torch.Tensor, handle: int) -> torch.Tensor:
    op, _ = _entry(handle, x)
    return op.forward_silu_mul(x, g)


@forward_silu_mul.register_fake
def _(x, g, handle):
    _, d_out = _entry(handle, x)
    return x.new_empty((x.shape[0], d_out))


@torch.library.custom_op("trring::consume_silu_mul", mutates_args=("g", "u"))
def consume_silu_mul(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    return _consume_silu_mul(g, u)


@consume_silu_mul.register_fake
def _(g, u):
    return g.new_empty(g.shape, dtype=torch.bfloat16)


@torch.library.custom_op("trring::consume_add", mutates_args=("y",))
def consume_add(h: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    return _consume_add(h, y)


@consume_add.register_fake
def _(h, y):
    return torch.empty_like(h)


@torch.library.custom_op("trring::plan_step", mutates_args=("tables",))
def plan_step(lens: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, free: torch.Tensor,
              free_count: torch.Tensor, page_size: int, tokens: int) -> tuple[
                  torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                  torch.Tensor]:
    return binding().plan_step(lens, new, tables, free, free_count, page_size, tokens, apart=True)


@plan_step.register_fake
def _(lens, new, tables, free, free_count, page_size, tokens):
    R = lens.shape[0]
    return (lens.new_empty(tokens, dtype=torch.int64), lens.new_empty(tokens),
            lens.new_empty(R + 1), lens.new_empty(R), lens.new_empty(R), lens.new_empty(1))


@torch.library.custom_op("trring::append_kv", mutates_args=("k_pages", "v_pages"))
def append_kv(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              slots: torch.Tensor) -> None:
    _serve.append_kv(k, v, k_pages, v_pages, slots)


@append_kv.register_fake
def _(k, v, k_pages, v_pages, slots):
    return None


@torch.library.custom_op("trring::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    tables: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor,
                    scale: Optional[float] = None) -> tuple[torch.Tensor, torch.Tensor]:
    return _serve.paged_attention(q, k_pages, v_pages, tables, lens, starts, scale=scale,
                                  return_lse=True)


@paged_attention.register_fake
def _(q, k_pages, v_pages, tables, lens, starts, scale=None):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.custom_op("trring::residual_norm", mutates_args=())
def residual_norm(y: torch.Tensor, h: torch.Tensor, post: Optional[torch.Tensor],
                  pre: torch.Tensor, gate: Optional[torch.Tensor],
                  post_bias: Optional[torch.Tensor], pre_bias: Optional[torch.Tensor], kind: str,
                  eps: float, residual_scale: float,
                  branch_scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    return _serve.residual_norm(y, h, post=post, pre=pre, gate=gate, post_bias=post_bias,
                                pre_bias=pre_bias, kind=kind, eps=eps,
                                residual_scale=residual_scale, branch_scale=branch_scale)


@residual_norm.register_fake
def _(y, h, post, pre, gate, post_bias, pre_bias, kind, eps, residual_scale, branch_scale):
    return h.new_empty(h.shape), h.new_empty(h.shape)


@torch.library.custom_op("trring::sample_tokens", mutates_args=())
def sample_tokens(logits: torch.Tensor, noise: torch.Tensor, temperature: torch.Tensor,
                  top_k: Optional[torch.Tensor], top_p: Optional[torch.Tensor],
                  min_p: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    return binding().sample_tokens(logits, noise, temperature, top_k, top_p, min_p, apart=True)


@sample_tokens.register_fake
def _(logits, noise, temperature, top_k, top_p, min_p):
    R = logits.shape[0]
    return (logits.new_empty(R, dtype=torch.int64), logits.new_empty(R, dtype=torch.float32))
