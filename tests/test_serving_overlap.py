"""Outputs that overlap themselves or an input are refused through the C ABI (on the CPU: every check comes
before the device is touched; the pointers are never followed)."""
from __future__ import annotations

import ctypes

import pytest

from autokernel_b200 import _lib

N, H, HKV, D, P, S = 3, 4, 2, 64, 4, 8
TOKENS_Q, TOKENS_K = (H * D, D), (HKV * D, D)
CACHE = (HKV * S * D, S * D, D)
ROOM = 1 << 20                           # between two tensors


def _st(v):
    return (ctypes.c_int64 * len(v))(*v)


def _message():
    return _lib.load().ak_last_error().decode()


def attention(out=4 * ROOM, out_st=TOKENS_Q, q=ROOM, scale=0.1, n=N, ws=0):
    """The call with its workspace missing: refused for that when everything before it is right."""
    lists = 16
    rc = _lib.load().ak_paged_attention(q, 2 * ROOM, 3 * ROOM, out, lists, lists, lists, n, 1, H, HKV, D, P, S, 3, 3,
                                        _st(TOKENS_Q), _st(out_st), _st(CACHE), _st(CACHE), 1, scale, 2, None, ws, None)
    return rc, _message()


@pytest.mark.parametrize("out_st", [TOKENS_Q, (1000, 100), (D, N * D), (H * D + 8, D)])
def test_attention_outputs_apart_pass(out_st):
    rc, why = attention(out_st=out_st)
    assert rc == -1 and "workspace" in why


@pytest.mark.parametrize("out_st", [(0, D), (H * D, 0), (H * D - 8, D), (H * D, D - 8), (D, D)])
def test_attention_outputs_that_overlap_themselves(out_st):
    rc, why = attention(out_st=out_st)
    assert rc == -1 and "overlap" in why


@pytest.mark.parametrize("out", [1, 2, 3])
def test_attention_output_over_an_input(out):
    rc, why = attention(out=out * ROOM)
    assert rc == -1 and "overlap" in why


@pytest.mark.parametrize("scale", [2.4e38, 3e38])
def test_scales_that_overflow_in_log2(scale):
    """(scaled by log2 e they are infinite, and a score of 0 becomes NaN)"""
    rc, why = attention(scale=scale, n=0)
    assert rc == -1 and "sm_scale" in why


def append(q_out=6 * ROOM, out_st=TOKENS_Q, kc_st=CACHE, vc_st=CACHE, k_cache=4 * ROOM, v_cache=5 * ROOM, q=3 * ROOM):
    rc = _lib.load().ak_paged_append(ROOM, 2 * ROOM, q, q_out, k_cache, v_cache, 16, 16, 16, 16, 16, N, 1, H, HKV, D,
                                     P, S, 3, 3, 9, _st(TOKENS_K), _st(TOKENS_K), _st(TOKENS_Q), _st(out_st),
                                     _st(kc_st), _st(vc_st), 2, None)
    return rc, _message()


@pytest.mark.parametrize("bad", [dict(out_st=(0, D)), dict(out_st=(H * D, 0)), dict(kc_st=(0, S * D, D)),
                                 dict(vc_st=(HKV * S * D, 0, D)), dict(kc_st=(HKV * S * D, S * D, 0)),
                                 dict(vc_st=(HKV * S * D - 8, S * D, D)), dict(v_cache=4 * ROOM), dict(q_out=ROOM),
                                 dict(q_out=2 * ROOM), dict(q_out=4 * ROOM), dict(q_out=3 * ROOM, out_st=(1000, D))])
def test_append_over_itself_or_an_input(bad):
    rc, why = append(**bad)
    assert rc == -1 and "overlap" in why
