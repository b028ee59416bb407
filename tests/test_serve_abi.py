"""CPU: the serving entry points of the C ABI refuse bad arguments before any launch."""
from __future__ import annotations

import ctypes
from ctypes import c_size_t

import pytest

from kernel_task_b200 import abi

P = 4096  # a non-null, 16-byte aligned address that is never followed


def attention(**over):
    a = abi.TrAttention(q=P, q_token_stride=512, q_head_stride=128, k_pages=P, v_pages=P, tables=P,
                        table_stride=4, lens=P, starts=P, out=P, lse=None, tokens=2, requests=2,
                        pages=9, columns=4, page_size=16, heads=4, kv_heads=2, head_dim=128,
                        dtype=abi.TR_BF16, scale=0.1)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(dtype=9), abi.TR_ERR_INVALID), (dict(heads=5), abi.TR_ERR_INVALID),
    (dict(kv_heads=0), abi.TR_ERR_INVALID), (dict(tokens=-1), abi.TR_ERR_INVALID),
    (dict(table_stride=3), abi.TR_ERR_INVALID), (dict(scale=0.0), abi.TR_ERR_INVALID),
    (dict(scale=float("nan")), abi.TR_ERR_INVALID), (dict(scale=float("inf")), abi.TR_ERR_INVALID),
    (dict(q=None), abi.TR_ERR_INVALID), (dict(lens=None), abi.TR_ERR_INVALID),
    (dict(tables=None), abi.TR_ERR_INVALID), (dict(v_pages=None), abi.TR_ERR_INVALID),
    (dict(q=P + 2), abi.TR_ERR_ALIGN), (dict(q_head_stride=65), abi.TR_ERR_ALIGN),
    (dict(head_dim=12), abi.TR_ERR_UNSUPPORTED), (dict(head_dim=264), abi.TR_ERR_UNSUPPORTED),
    (dict(page_size=24), abi.TR_ERR_UNSUPPORTED), (dict(page_size=2048), abi.TR_ERR_UNSUPPORTED),
    (dict(columns=1 << 28, table_stride=1 << 28), abi.TR_ERR_UNSUPPORTED),
])
def test_attention_arguments(over, status):
    a = attention(**over)
    assert abi.lib().tr_paged_attention(ctypes.byref(a), None, 0, None) == status
    assert abi.lib().tr_last_error()
    n = c_size_t()
    assert abi.lib().tr_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == status


def test_attention_of_no_tokens():
    a = attention(tokens=0, q=None, out=None, k_pages=None, v_pages=None)
    assert abi.lib().tr_paged_attention(ctypes.byref(a), None, 0, None) == abi.TR_OK
    assert abi.lib().tr_paged_attention(None, None, 0, None) == abi.TR_ERR_INVALID
    assert abi.lib().tr_attention_workspace_bytes(ctypes.byref(attention()), None) == \
        abi.TR_ERR_INVALID


def norm(**over):
    n = abi.TrNorm(y=P, h=P, gate=P, post=P, post_bias=None, pre=P, pre_bias=None, h_out=P, x_out=P,
                   tokens=3, width=64, y_stride=64, h_stride=64, gate_stride=0,
                   kind=abi.TR_NORM_RMS, dtype=abi.TR_BF16, y_dtype=abi.TR_F32, eps=1e-6,
                   residual_scale=1.0, branch_scale=1.0)
    for k, v in over.items():
        setattr(n, k, v)
    return n


@pytest.mark.parametrize("over,status", [
    (dict(dtype=3), abi.TR_ERR_INVALID), (dict(y_dtype=abi.TR_F16), abi.TR_ERR_INVALID),
    (dict(kind=2), abi.TR_ERR_INVALID), (dict(width=0), abi.TR_ERR_INVALID),
    (dict(tokens=-1), abi.TR_ERR_INVALID), (dict(width=32769), abi.TR_ERR_UNSUPPORTED),
    (dict(y=None), abi.TR_ERR_INVALID), (dict(y=None, post=None, gate=None, pre=None), abi.TR_ERR_INVALID),
    (dict(post=None, post_bias=P), abi.TR_ERR_INVALID), (dict(h=None), abi.TR_ERR_INVALID),
    (dict(h_out=None), abi.TR_ERR_INVALID), (dict(x_out=None), abi.TR_ERR_INVALID),
    (dict(eps=-1.0), abi.TR_ERR_INVALID), (dict(eps=float("nan")), abi.TR_ERR_INVALID),
    (dict(h=P + 1), abi.TR_ERR_ALIGN), (dict(y=P + 2), abi.TR_ERR_ALIGN),
])
def test_norm_arguments(over, status):
    assert abi.lib().tr_residual_norm(ctypes.byref(norm(**over)), None) == status
    assert abi.lib().tr_residual_norm(ctypes.byref(norm(tokens=0)), None) == abi.TR_OK
    assert abi.lib().tr_residual_norm(None, None) == abi.TR_ERR_INVALID


def test_sample_arguments():
    call = abi.lib().tr_sample
    good = [P, abi.TR_F32, 100, P, 100, P, P, P, P, 2, 100, P, P, None]
    for at, value, status in [(0, None, abi.TR_ERR_INVALID), (1, 5, abi.TR_ERR_INVALID),
                              (3, None, abi.TR_ERR_INVALID), (5, None, abi.TR_ERR_INVALID),
                              (11, None, abi.TR_ERR_INVALID), (9, -1, abi.TR_ERR_INVALID),
                              (10, 0, abi.TR_ERR_INVALID), (10, (1 << 22) + 1, abi.TR_ERR_UNSUPPORTED),
                              (0, P + 2, abi.TR_ERR_ALIGN), (11, P + 4, abi.TR_ERR_ALIGN)]:
        args = list(good)
        args[at] = value
        assert call(*args) == status, (at, value)
    args = list(good)
    args[9] = 0
    assert call(*args) == abi.TR_OK


def test_step_and_append_arguments():
    lib = abi.lib()
    good = [P, P, 4, P, 8, 8, P, 100, P, 16, 64, P, P, P, P, P, P, None]
    for at, value, status in [(0, None, abi.TR_ERR_INVALID), (2, -1, abi.TR_ERR_INVALID),
                              (2, 16385, abi.TR_ERR_UNSUPPORTED), (3, None, abi.TR_ERR_INVALID),
                              (4, 7, abi.TR_ERR_INVALID), (6, None, abi.TR_ERR_INVALID),
                              (7, 1 << 31, abi.TR_ERR_INVALID), (8, None, abi.TR_ERR_INVALID),
                              (9, 0, abi.TR_ERR_INVALID), (10, -1, abi.TR_ERR_INVALID),
                              (10, 1 << 31, abi.TR_ERR_INVALID), (11, None, abi.TR_ERR_INVALID),
                              (13, None, abi.TR_ERR_INVALID), (16, None, abi.TR_ERR_INVALID)]:
        args = list(good)
        args[at] = value
        assert lib.tr_plan_step(*args) == status, (at, value)
    good = [P, P, 4, P, 8, 8, P, 100, P, 16, None]
    for at, value, status in [(1, None, abi.TR_ERR_INVALID), (2, 16385, abi.TR_ERR_UNSUPPORTED),
                              (9, 0, abi.TR_ERR_INVALID), (2, 0, abi.TR_OK)]:
        args = list(good)
        args[at] = value
        assert lib.tr_release_pages(*args) == status, (at, value)
    good = [P, 128, 64, P, 128, 64, abi.TR_BF16, P, P, abi.TR_BF16, P, 3, 2, 64, 10, 16, None]
    for at, value, status in [(0, None, abi.TR_ERR_INVALID), (6, abi.TR_F16, abi.TR_ERR_INVALID),
                              (9, 7, abi.TR_ERR_INVALID), (7, P + 2, abi.TR_ERR_ALIGN),
                              (0, P + 1, abi.TR_ERR_ALIGN), (10, P + 4, abi.TR_ERR_ALIGN),
                              (12, 0, abi.TR_ERR_INVALID), (15, 0, abi.TR_ERR_INVALID),
                              (11, 0, abi.TR_OK), (14, 0, abi.TR_OK)]:
        args = list(good)
        args[at] = value
        assert lib.tr_append_kv(*args) == status, (at, value)


@pytest.mark.parametrize("name", ["tables", "lens", "starts", "lse"])
def test_attention_index_pointers_off_their_elements(name):
    a = attention(**{name: P + 2})
    assert abi.lib().tr_paged_attention(ctypes.byref(a), None, 0, None) == abi.TR_ERR_ALIGN


def test_attention_of_more_tokens_than_an_index_holds():
    # their product with the heads passes 64 bits
    a = attention(tokens=1 << 62)
    assert abi.lib().tr_paged_attention(ctypes.byref(a), None, 0, None) == abi.TR_ERR_UNSUPPORTED


def test_step_pointers_off_their_elements():
    lib = abi.lib()
    good = [P, P, 4, P, 8, 8, P, 100, P, 16, 64, P, P, P, P, P, P, None]
    for at in (0, 1, 3, 6, 8, 12, 13, 14, 15, 16):
        assert lib.tr_plan_step(*good[:at], P + 2, *good[at + 1:]) == abi.TR_ERR_ALIGN, at
    assert lib.tr_plan_step(*good[:11], P + 4, *good[12:]) == abi.TR_ERR_ALIGN
    good = [P, P, 4, P, 8, 8, P, 100, P, 16, None]
    for at in (0, 1, 3, 6, 8):
        assert lib.tr_release_pages(*good[:at], P + 2, *good[at + 1:]) == abi.TR_ERR_ALIGN, at
