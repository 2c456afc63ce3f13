"""What the serving operators refuse, checked on CPU tensors and through the C ABI (every check
comes before the device is touched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from autokernel_b200 import _lib, ops

I32 = torch.int32


def _cache(P=4, Hkv=2, S=8, D=64, dt=torch.bfloat16):
    return torch.zeros(P, Hkv, S, D, dtype=dt), torch.zeros(P, Hkv, S, D, dtype=dt)


def _args(**kw):
    kc, vc = _cache()
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
             v=torch.zeros(3, 2, 64, dtype=torch.bfloat16), k_cache=kc, v_cache=vc,
             page_table=torch.zeros(2, 3, dtype=I32), cu_q=torch.tensor([0, 1, 3], dtype=I32),
             kv_lens=torch.tensor([5, 6], dtype=I32), cos=torch.zeros(9, 32), sin=torch.zeros(9, 32))
    a.update(kw)
    return a


def _attend(a, **kw):
    return ops.paged_attention(a["q"], a["k_cache"], a["v_cache"], a["page_table"], a["cu_q"], a["kv_lens"], **kw)


def _append(a, **kw):
    return ops.paged_append(a["k"], a["v"], a["k_cache"], a["v_cache"], a["page_table"], a["cu_q"],
                            a["kv_lens"], q=a["q"], cos=a["cos"], sin=a["sin"], **kw)


BAD_LISTS = [
    dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), dict(cu_q=torch.zeros(3)),
    dict(kv_lens=torch.zeros(2, dtype=torch.int64)), dict(page_table=torch.zeros(3, 3, dtype=I32)),
    dict(cu_q=torch.zeros(2, dtype=I32)), dict(kv_lens=torch.zeros(2, 1, dtype=I32)),
    dict(page_table=torch.zeros(2, 6, dtype=I32)[:, ::2]), dict(cu_q=torch.zeros(6, dtype=I32)[::2]),
    dict(v_cache=torch.zeros(4, 2, 8, 32, dtype=torch.bfloat16)),
    dict(v_cache=torch.zeros(4, 2, 8, 64, dtype=torch.float16)),
    dict(k_cache=torch.zeros(4, 2, 64, 8, dtype=torch.bfloat16).transpose(2, 3)),
    dict(k_cache=torch.zeros(4, 2, 0, 64, dtype=torch.bfloat16), v_cache=torch.zeros(4, 2, 0, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(3, 4 * 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
]


@pytest.mark.parametrize("bad", BAD_LISTS, ids=range(len(BAD_LISTS)))
def test_bad_cache_lists_and_queries(bad):
    with pytest.raises(ValueError, match="paged_attention"):
        _attend(_args(**bad))
    with pytest.raises(ValueError, match="paged_append"):
        _append(_args(**bad))


def test_attention_refusals():
    with pytest.raises(ValueError, match="multiple"):
        _attend(_args(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)))
    for s in (0.0, -0.1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="sm_scale"):
            _attend(_args(), sm_scale=s)
    kc, vc = _cache(D=264)
    with pytest.raises(ValueError, match="256"):
        _attend(_args(q=torch.zeros(3, 4, 264, dtype=torch.bfloat16), k_cache=kc, v_cache=vc))
    with pytest.raises(ValueError, match="out"):
        _attend(_args(), out=torch.zeros(3, 2, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        _attend(_args())
    kc, vc = (c.double() for c in _cache())
    with pytest.raises(ValueError, match="dtype"):
        _attend(_args(q=torch.zeros(3, 4, 64, dtype=torch.float64), k_cache=kc, v_cache=vc))


def test_append_refusals():
    bad = [dict(k=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), dict(v=torch.zeros(2, 2, 64, dtype=torch.bfloat16)),
           dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), dict(cos=None), dict(cos=None, sin=None),
           dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64)), dict(cos=torch.zeros(9, 32).half()),
           dict(cos=torch.zeros(9, 64)[:, ::2]), dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)),
           dict(cos=torch.zeros(9, 2, 32), sin=torch.zeros(9, 2, 32))]
    for b in bad:
        with pytest.raises(ValueError, match="paged_append"):
            _append(_args(**b))
    with pytest.raises(ValueError, match="q_out without q"):
        _append(_args(q=None), q_out=torch.zeros(3, 4, 64, dtype=torch.bfloat16))
    kc, vc = _cache(D=7)
    t = torch.zeros(3, 2, 7, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="even"):
        _append(_args(k=t, v=t, q=None, cos=None, sin=None, k_cache=kc, v_cache=vc))
    with pytest.raises(ValueError, match="CUDA"):
        _append(_args())


def test_sample_refusals():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=float("nan")), dict(min_p=-0.1),
                dict(temperature=torch.ones(2)), dict(top_k=torch.ones(3)), dict(top_p=torch.ones(3).double())):
        with pytest.raises(ValueError, match="sample"):
            ops.sample(x, u, **bad)
    for args in ((x[0], u), (x[:, :0], u), (x, u[:2]), (x, u.double()), (x.int(), u)):
        with pytest.raises(ValueError):
            ops.sample(*args)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample(x, u)


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _abi_attention(H=4, Hkv=2, D=64, S=8, scale=0.1, dt=2, N=3, B=1, ws=1 << 40, q=16):
    s2, s3 = _st(H * D, D), _st(Hkv * S * D, S * D, D)
    return _lib.load().ak_paged_attention(q, 16, 16, 16, 16, 16, 16, N, B, H, Hkv, D, 4, S, 3, 3, s2, s2, s3, s3,
                                          1, scale, dt, 16, ws, None)


@pytest.mark.parametrize("kw,code", [(dict(dt=5), -2), (dict(H=3), -3), (dict(D=0), -3), (dict(D=264), -3),
                                     (dict(S=0), -3), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
                                     (dict(ws=0), -1), (dict(q=None), -1), (dict(N=-1), -3),
                                     (dict(N=0), 0), (dict(B=0), 0)])
def test_abi_attention(kw, code):
    assert _abi_attention(**kw) == code
    assert code == 0 or _lib.load().ak_last_error()


def _abi_append(D=64, cos=16, sin=16, positions=9, q=16, q_out=16, dt=2, N=3, k=16):
    s2, s3 = _st(2 * D, D), _st(2 * 8 * D, 8 * D, D)
    return _lib.load().ak_paged_append(k, 16, q, q_out, 16, 16, 16, 16, 16, cos, sin, N, 1, 4, 2, D, 4, 8, 3, 3,
                                       positions, s2, s2, s2, s2, s3, s3, dt, None)


@pytest.mark.parametrize("kw,code", [(dict(dt=3), -2), (dict(D=7), -3), (dict(D=0), -3), (dict(cos=None), -1),
                                     (dict(positions=0), -3), (dict(q_out=None), -1), (dict(k=None), -1),
                                     (dict(N=0), 0)])
def test_abi_append(kw, code):
    assert _abi_append(**kw) == code


def _abi_sample(rows=2, vocab=10, ld=10, dt=2, x=16, out=16):
    return _lib.load().ak_sample(x, 16, rows, vocab, ld, dt, None, None, None, None, 1.0, 0, 1.0, 0.0, out, None)


@pytest.mark.parametrize("kw,code", [(dict(dt=9), -2), (dict(vocab=0), -3), (dict(ld=-1), -3), (dict(rows=-1), -3),
                                     (dict(x=None), -1), (dict(out=None), -1), (dict(rows=0), 0)])
def test_abi_sample(kw, code):
    assert _abi_sample(**kw) == code
