"""The serving operators (ops.paged_append, ops.paged_attention, ops.sample) against their float64
restatement (oracle/serve_f64.py).

Bounds, derived from the arithmetic (h = half a step of the output type relative to the value):
  append     h |e| + 3 * 2^-24 (|x1 c| + |x2 s|): two fp32 products, one sum, one rounding; without a
             rotation, values and keys are copies and have to be equal.
  attention  with A = softmax . |V| and d = (D + 8) 2^-24 max_j scale sum |q||k_j| + 2^-20 (the fp32
             dot product, the product with the scale, the exponential): every weight is off by a
             factor 1 +- 2 d, weights are rounded to 16 bits once (h; not in fp32), and the sums over
             L keys are fp32 in any order (L 2^-24), so |y - e| <= h |e| + (h + 2 d + (L + 8) 2^-23) A.
  sample     tokens are equal.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from autokernel_b200 import ops
from oracle import serve_f64

pytestmark = pytest.mark.gpu

DTS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def _half(dt):
    return torch.finfo(dt).eps / 2


def n64(t):
    return t.detach().double().cpu().numpy()


class Batch:
    """A cache filled with stale values and the lists of sequences (new tokens, keys in all)."""

    def __init__(self, dt, seqs, kv_heads, D, page, seed=0, rows_behind=0, layout="pages",
                 stale=None, spare=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.g, self.dt, self.D, self.Hkv = g, DTS[dt], D, kv_heads
        new, lens = [s[0] for s in seqs], [s[1] for s in seqs]
        used = [-(-x // page) for x in lens]
        P = sum(used) + spare
        perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((len(seqs), max(used + [1]) + 1), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = perm[at:at + n]
            at += n
        self.table = table.to(DEV)
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.N = sum(new) + rows_behind
        if layout == "slots":  # [P, S, Hkv, D] seen as [P, Hkv, S, D]
            make = lambda: self.normal(P, page, kv_heads, D).transpose(1, 2)  # noqa: E731
        elif layout == "padded":
            make = lambda: self.normal(P, kv_heads, page, D + 8)[..., :D]  # noqa: E731
        else:
            make = lambda: self.normal(P, kv_heads, page, D)  # noqa: E731
        self.kc, self.vc = make(), make()
        if stale is not None:  # every slot that no sequence owns holds this
            own = torch.zeros(P, page, dtype=torch.bool)
            for b, n in enumerate(lens):
                for j in range(n):
                    own[table[b, j // page], j % page] = True
            own = own.to(DEV)[:, None, :, None]
            for c in (self.kc, self.vc):
                c.copy_(torch.where(own, c, torch.full_like(c, stale)))

    def normal(self, *shape):
        return torch.randn(*shape, device=DEV, generator=self.g).to(self.dt)

    def lists(self):
        return self.table, self.cu, self.lens

    def host_lists(self):
        return tuple(t.cpu().numpy() for t in self.lists())


def check_attention(b: Batch, q, out, causal=True, scale=None, rows=None):
    scale = b.D ** -0.5 if scale is None else scale
    e, A, spread, live = serve_f64.paged_attention(n64(q), n64(b.kc), n64(b.vc), *b.host_lists(), causal, scale)
    y, h = n64(out), _half(b.dt)
    L = max(b.lens.tolist() + [1])
    d = (b.D + 8) * 2.0 ** -24 * spread + 2.0 ** -20
    tol = h * np.abs(e) + ((0 if b.dt == torch.float32 else h) + 2 * d + (L + 8) * 2.0 ** -23) * A
    live = live if rows is None else live & rows
    assert live.any()
    nan = np.isnan(e[live])
    assert np.array_equal(np.isnan(y[live]), nan)
    err = np.where(nan, 0, np.abs(y[live] - e[live]) - tol[live])
    assert not (err > 0).any(), (float(err.max()), np.argwhere(err > 0)[:4])


def attend(b: Batch, heads, causal=True, scale=None, out=None, q=None):
    q = b.normal(b.N, heads, b.D) if q is None else q
    o = ops.paged_attention(q, b.kc, b.vc, *b.lists(), causal=causal, sm_scale=scale, out=out)
    torch.cuda.synchronize()
    return q, o


# ------------------------------------------------------------------------------------ append

def tables(positions, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(positions, dtype=torch.float64), inv)
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


def check_append(b: Batch, k, v, q, cos, sin, run):
    kc0, vc0, q0 = n64(b.kc), n64(b.vc), n64(q) if q is not None else None
    cs = (n64(cos), n64(sin)) if cos is not None else (None, None)
    ek, ev, eq = serve_f64.paged_append(n64(k), n64(v), kc0, vc0, *b.host_lists(), q0, *cs)
    got_q = run()
    torch.cuda.synchronize()
    assert np.array_equal(n64(b.vc), ev, equal_nan=True)
    if cos is None:
        assert np.array_equal(n64(b.kc), ek, equal_nan=True)
        return got_q
    h = _half(b.dt)

    def near(y, e, most):
        assert np.array_equal(np.isnan(y), np.isnan(e))
        err = np.abs(y - e) - (h * np.abs(e) + 3 * 2.0 ** -24 * 2 * most)
        assert not (err > 0).any(), float(np.nanmax(err))

    near(n64(b.kc), ek, np.abs(n64(k)).max())
    untouched = ek == kc0
    assert np.array_equal(n64(b.kc)[untouched], kc0[untouched])
    if q is not None:
        places = serve_f64.token_places(*b.host_lists(), b.N, kc0.shape[0], kc0.shape[2])
        live = np.array([w is not None for w in places])
        near(n64(got_q)[live], eq[live], np.abs(q0).max())
    return got_q


RAGGED = [(1, 1), (0, 40), (7, 23), (1, 129), (16, 16), (0, 0), (3, 64)]


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("heads,kv,D,page,layout", [(4, 4, 128, 16, "pages"), (6, 2, 64, 24, "slots"),
                                                    (3, 1, 80, 5, "pages"), (2, 2, 6, 3, "padded"),
                                                    (32, 8, 128, 64, "padded"), (1, 1, 256, 1, "pages")])
def test_append_ragged(dt, heads, kv, D, page, layout):
    b = Batch(dt, RAGGED, kv, D, page, seed=D + page, rows_behind=5, layout=layout)
    k, v, q = b.normal(b.N, kv, D), b.normal(b.N, kv, D), b.normal(b.N, heads, D)
    cos, sin = tables(200, D)
    check_append(b, k, v, q, cos, sin,
                 lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists(), q=q, cos=cos, sin=sin))


@pytest.mark.parametrize("dt", list(DTS))
def test_append_without_rotation_copies(dt):
    b = Batch(dt, RAGGED, 2, 64, 16, seed=1)
    k, v = b.normal(b.N, 2, 64), b.normal(b.N, 2, 64)
    assert check_append(b, k, v, None, None, None,
                        lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists())) is None


@pytest.mark.parametrize("dt", list(DTS))
def test_append_from_a_fused_projection_in_place(dt):
    """q, k, v are views of one row; q is rotated where it lies and its neighbours stay."""
    b = Batch(dt, RAGGED, 2, 64, 16, seed=2, rows_behind=3)
    qkv = b.normal(b.N, 10, 64)
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    before = qkv.clone()
    cos, sin = tables(200, 64)
    got = check_append(b, k, v, q, cos, sin,
                       lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists(), q=q, cos=cos[:, None],
                                                sin=sin[:, None], q_out=q))
    assert got is q
    assert torch.equal(qkv[:, 6:], before[:, 6:])
    assert torch.equal(qkv[int(b.cu[-1]):], before[int(b.cu[-1]):])  # rows behind the last sequence


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_unaligned_views(dt):
    """An odd element offset rules out 16-byte accesses."""
    b = Batch(dt, RAGGED, 2, 64, 16, seed=3)
    flat = b.normal(b.N * 2 * 65 + 1)
    k = flat[1:1 + b.N * 130].view(b.N, 2, 65)[..., :64]
    v, q = b.normal(b.N, 2, 64), b.normal(b.N, 4, 64)
    cos, sin = (x.flatten().clone() for x in tables(200, 64))
    check_append(b, k, v, q, cos.view(200, 32), sin.view(200, 32),
                 lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists(), q=q, cos=cos.view(200, 32),
                                          sin=sin.view(200, 32)))


@pytest.mark.parametrize("D", [64, 10])
def test_append_bad_places(D):
    """Pages outside the cache, positions outside the table row, negative positions and positions
    outside the rotation tables store nothing, or NaN where no angle is known."""
    b = Batch("f16", [(4, 40), (5, 3), (2, 64), (3, 30)], 2, D, 16, seed=4)
    b.table[0, 2] = b.kc.shape[0]          # one behind the last page
    b.table[2, 3] = -1
    b.table = b.table[:, :4].contiguous()
    b.lens[2] = 65                         # its last key lies behind the table row
    k, v, q = b.normal(b.N, 2, D), b.normal(b.N, 2, D), b.normal(b.N, 2, D)
    cos, sin = tables(29, D)               # sequence 3 writes positions 27..29
    check_append(b, k, v, q, cos, sin,
                 lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists(), q=q, cos=cos, sin=sin))


def test_append_clamps_token_ranges():
    """cu_q entries outside [0, N] or descending name no token."""
    b = Batch("bf16", [(4, 40), (5, 9)], 1, 64, 16, seed=5)
    k, v = b.normal(b.N, 1, 64), b.normal(b.N, 1, 64)
    kc, vc = b.kc.clone(), b.vc.clone()
    for cu in ([0, 2 ** 31 - 1, -5], [-2 ** 31, -1, -1], [b.N, b.N + 1, 2 ** 31 - 1], [6, 3, 0]):
        b.cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        b.lens = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
        ops.paged_append(k, v, b.kc, b.vc, *b.lists())
    torch.cuda.synchronize()
    assert torch.equal(b.kc, kc) and torch.equal(b.vc, vc)


# ------------------------------------------------------------------------------------ attention

SHAPES = [(4, 4, 128, 16), (8, 2, 64, 64), (6, 1, 128, 24), (32, 8, 128, 8), (16, 1, 64, 128),
          (20, 1, 128, 16), (12, 12, 64, 256), (7, 7, 64, 40), (3, 1, 80, 16), (2, 1, 256, 16),
          (4, 2, 64, 5), (2, 2, 10, 1)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("heads,kv,D,page", SHAPES)
def test_attention_ragged(dt, heads, kv, D, page, causal):
    b = Batch(dt, [(1, 1), (0, 40), (7, 23), (1, 300), (40, 40), (0, 0), (3, 64), (1, 65)], kv, D, page,
              seed=heads * D + page, rows_behind=2, stale=float("nan"))
    q, o = attend(b, heads, causal)
    check_attention(b, q, o, causal)


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("heads,kv,D,page", [(4, 4, 128, 16), (8, 2, 64, 64), (8, 1, 128, 24)])
def test_attention_decode(dt, heads, kv, D, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 2049]
    b = Batch(dt, [(1, x) for x in lens], kv, D, page, seed=D, stale=float("inf"))
    q, o = attend(b, heads)
    check_attention(b, q, o)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,D,page,seqs", [
    (2, 2, 128, 64, [(300, 300), (129, 700), (1, 513), (64, 64)]),
    (8, 2, 64, 16, [(257, 1000), (5, 5), (200, 201)]),
    (5, 1, 128, 48, [(150, 150), (33, 400)]),
    (64, 1, 64, 128, [(9, 140), (3, 3)]),
    (1, 1, 128, 128, [(513, 513)]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_chunks(dt, heads, kv, D, page, seqs, causal):
    b = Batch(dt, seqs, kv, D, page, seed=D + page, stale=float("nan"))
    q, o = attend(b, heads, causal)
    check_attention(b, q, o, causal)


@pytest.mark.parametrize("layout", ["slots", "padded"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_attention_strided_cache_and_tokens(dt, layout):
    b = Batch(dt, [(1, 90), (70, 200)], 2, 64, 16, seed=9, layout=layout)
    wide = b.normal(b.N, 12, 64)
    q = wide[:, 2:10]
    store = torch.full((b.N + 2, 9, 72), 7.0, device=DEV, dtype=b.dt)
    out = store[1:-1, :8, :64]
    got = ops.paged_attention(q, b.kc, b.vc, *b.lists(), out=out)
    torch.cuda.synchronize()
    assert got is out
    check_attention(b, q, out)
    store[1:-1, :8, :64] = 7.0
    assert (store == 7.0).all()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_attention_unaligned_views(dt):
    b = Batch(dt, [(1, 90), (30, 100)], 1, 64, 16, seed=10)
    flat = b.normal(b.N * 2 * 65 + 1)
    q = flat[1:].view(b.N, 2, 65)[..., :64]
    o = torch.empty(b.N * 2 * 65 + 1, device=DEV, dtype=b.dt)[1:].view(b.N, 2, 65)[..., :64]
    attend(b, 2, q=q, out=o)
    check_attention(b, q, o)
    kv = b.normal(b.kc.numel() + 1)
    b.kc = kv[1:].view(b.kc.shape)
    q, o = attend(b, 2)
    check_attention(b, q, o)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_rows_without_keys_are_zero(dt, D):
    """Fewer keys than new tokens: the first rows sit at negative positions and see nothing."""
    b = Batch(dt, [(5, 3), (1, 0), (200, 150), (2, 0)], 2, D, 16, seed=11, stale=float("nan"))
    for causal in (True, False):
        q, o = attend(b, 4, causal, out=torch.full((b.N, 4, D), 3.0, device=DEV, dtype=b.dt))
        check_attention(b, q, o, causal)
        assert (o[5] == 0).all() and (o[-2:] == 0).all()
    assert (attend(b, 4)[1][:2] == 0).all()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_attention_missing_pages_give_nan_where_they_are_seen(dt):
    b = Batch(dt, [(40, 40), (1, 100), (150, 300), (1, 33), (3, 50)], 2, 64, 16, seed=12, stale=float("nan"))
    b.table[0, 1] = -1                      # seen from position 16 on
    b.table[1, 6] = b.kc.shape[0]           # the only row sees it
    b.table[2, 17] = 2 ** 31 - 1            # positions 272 and later
    b.lens[4] = 2 ** 31 - 1                 # far more keys than the table can name
    q, o = attend(b, 4)
    bad = n64(o)
    check_attention(b, q, o, rows=np.arange(b.N) < int(b.cu[4]))
    assert np.isnan(bad[16:40]).all() and not np.isnan(bad[:16]).any()
    assert np.isnan(bad[int(b.cu[4]):]).all()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,length", [(5, 30), (130, 200)])
def test_attention_hidden_keys_never_matter(dt, value, new, length):
    """A key that only later tokens see holds NaN or infinities: the earlier rows are as without it."""
    b = Batch(dt, [(new, length)], 1, 64, 16, seed=13)
    at = length - 3                          # seen by the last three tokens only
    page, slot = int(b.table[0, at // 16]), at % 16
    b.kc[page, :, slot] = value
    b.vc[page, :, slot] = value
    q, o = attend(b, 2)
    check_attention(b, q, o)
    assert o[:-3].isfinite().all() and o[-3:].isnan().all()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_attention_large_scores(dt):
    """Scores of thousands: the running maximum keeps the exponentials in range."""
    b = Batch(dt, [(1, 200), (140, 260)], 1, 64, 16, seed=14)
    q = b.normal(b.N, 2, 64) * 64
    b.kc *= 16
    _, o = attend(b, 2, q=q)
    assert o.isfinite().all()
    check_attention(b, q, o)


def test_attention_rows_behind_the_last_sequence_stay():
    for seqs in ([(1, 20), (1, 9)], [(140, 140), (2, 50)]):
        b = Batch("bf16", seqs, 2, 128, 16, seed=15, rows_behind=200)
        out = torch.full((b.N, 4, 128), 5.0, device=DEV, dtype=b.dt)
        q, _ = attend(b, 4, out=out)
        n = int(b.cu[-1])
        check_attention(b, q, out)
        assert (out[n:] == 5.0).all()


def test_offsets_past_32_bits():
    """Pages whose element offsets exceed 2^32."""
    D, Hkv, page = 128, 8, 32
    P = 2 ** 32 // (Hkv * page * D) + 200
    k = torch.empty(P, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    b = Batch("bf16", [(1, 70), (130, 150)], Hkv, D, page, seed=16)
    far = torch.arange(b.kc.shape[0], device=DEV) + (P - b.kc.shape[0])
    k[far], v[far] = b.kc, b.vc
    table = torch.where(b.table >= 0, b.table + (P - b.kc.shape[0]), b.table).int()
    q = b.normal(b.N, 16, D)
    nk, nv = b.normal(b.N, Hkv, D), b.normal(b.N, Hkv, D)
    cos, sin = tables(200, D)
    q1 = ops.paged_append(nk, nv, k, v, table, b.cu, b.lens, q=q, cos=cos, sin=sin)
    q2 = ops.paged_append(nk, nv, b.kc, b.vc, *b.lists(), q=q, cos=cos, sin=sin)
    assert torch.equal(q1, q2) and torch.equal(k[far], b.kc) and torch.equal(v[far], b.vc)
    o1 = ops.paged_attention(q1, k, v, table, b.cu, b.lens)
    o2 = ops.paged_attention(q2, b.kc, b.vc, *b.lists())
    assert torch.equal(o1, o2)
    check_attention(b, q2, o2)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_is_deterministic_and_keeps_its_inputs(dt):
    b = Batch(dt, [(1, 4000), (200, 900), (1, 3)], 2, 128, 16, seed=17)
    kc, vc = b.kc.clone(), b.vc.clone()
    q, o = attend(b, 8)
    q0 = q.clone()
    for _ in range(3):
        assert torch.equal(attend(b, 8, q=q)[1], o)
    assert torch.equal(b.kc, kc) and torch.equal(b.vc, vc) and torch.equal(q, q0)


def test_empty_calls():
    b = Batch("bf16", [(1, 5)], 1, 64, 16)
    none = torch.empty(0, 1, 64, device=DEV, dtype=b.dt)
    assert ops.paged_attention(none, b.kc, b.vc, *b.lists()).shape == (0, 1, 64)
    assert ops.paged_append(none, none, b.kc, b.vc, *b.lists()) is None
    q = torch.ones(2, 1, 64, device=DEV, dtype=b.dt)
    out = torch.full_like(q, 4.0)
    ops.paged_attention(q, b.kc, b.vc, b.table[:0], b.cu[:1], b.lens[:0], out=out)
    assert (out == 4).all()
    assert ops.sample(torch.empty(0, 5, device=DEV), torch.empty(0, device=DEV)).shape == (0,)


# ------------------------------------------------------------------------------------ sample

def check_sample(x, u, **kw):
    got = ops.sample(x, u, **kw).cpu().tolist()
    xs, us = n64(x), u.cpu().tolist()

    def at(name, r):
        v = kw.get(name, {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}[name])
        return v[r].item() if isinstance(v, torch.Tensor) else float(np.float32(v)) if name != "top_k" else v

    want = [serve_f64.sample_row(xs[r], us[r], *(at(n, r) for n in ("temperature", "top_k", "top_p", "min_p")))
            for r in range(x.shape[0])]
    assert got == want, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w][:5]


def logits(dt, rows, vocab, seed, scale=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab, device=DEV, generator=g) * scale
    return x.to(DTS[dt]), torch.rand(rows, device=DEV, generator=g)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3, top_k=1), dict(top_k=50),
            dict(temperature=1.3, top_k=7, top_p=0.8), dict(top_p=0.9), dict(top_p=0.3, min_p=0.05),
            dict(min_p=0.1), dict(temperature=2.0, top_k=3000, top_p=0.97, min_p=0.001),
            dict(top_p=0.0), dict(min_p=1.0), dict(min_p=7.0), dict(top_k=10 ** 9),
            dict(temperature=0.02, top_p=0.5), dict(temperature=1e30), dict(top_p=1e-30)]


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
def test_sample_settings(dt, kw):
    for vocab in (1000, 32000):
        check_sample(*logits(dt, 24, vocab, vocab), **kw)


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 31, 33, 255, 256, 257, 1023, 4097, 8191, 50257, 131072, 200001])
def test_sample_sizes(dt, vocab):
    x, u = logits(dt, 5, vocab, vocab + 1)
    for kw in (dict(), dict(top_k=5), dict(top_p=0.9), dict(top_k=40, top_p=0.9, min_p=0.02)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", list(DTS))
def test_sample_settings_per_row(dt):
    rows = 160
    x, u = logits(dt, rows, 5000, 3)
    g = torch.Generator(device=DEV).manual_seed(4)
    r = torch.rand(4, rows, device=DEV, generator=g)
    check_sample(x, u, temperature=torch.where(r[0] < 0.2, 0.0, 2 * r[0]),
                 top_k=torch.where(r[1] < 0.4, 0, 300 * r[1]).int(),
                 top_p=torch.where(r[2] < 0.3, 1.0, r[2]), min_p=torch.where(r[3] < 0.5, 0.0, 0.1 * r[3]))


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("temperature", [1e-30, 1e-4, 0.01, 0.1, 0.3, 0.49, 5.0, 100.0, float("inf")])
def test_sample_temperatures(dt, temperature):
    """Cuts among very uneven and very even weights."""
    x, u = logits(dt, 8, 40000, 10)
    for kw in (dict(top_p=0.6), dict(top_p=0.999), dict(top_k=20000, top_p=0.95), dict(min_p=0.5)):
        check_sample(x, u, temperature=temperature, **kw)


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("vocab", [262144, 262145, 300001])
def test_sample_longest_rows(dt, vocab):
    """Up to and beyond the rows that a cluster holds."""
    x, u = logits(dt, 3, vocab, vocab)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=900, top_p=0.5, min_p=0.01)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("levels", [1, 2, 5, 60])
def test_sample_ties(dt, levels):
    """Few distinct logits: cuts fall inside groups of equal ones, lowest index first."""
    g = torch.Generator(device=DEV).manual_seed(levels)
    x = (torch.randint(0, levels, (32, 3001), device=DEV, generator=g) * 0.25).to(DTS[dt])
    u = torch.rand(32, device=DEV, generator=g)
    for kw in (dict(), dict(top_k=10), dict(top_k=1500), dict(top_p=0.5), dict(top_p=0.1, top_k=2000),
               dict(min_p=0.6), dict(temperature=0.0), dict(top_k=1)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", list(DTS))
def test_sample_edges_of_u(dt):
    x, _ = logits(dt, 9, 700, 5)
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, float("nan"), 0.99999994, 1e-45, float("inf"), 0.5], device=DEV)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.7), dict(temperature=0.05)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", list(DTS))
def test_sample_infinities_and_nan(dt):
    x, u = logits(dt, 12, 1500, 6)
    inf, nan = float("inf"), float("nan")
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = nan
    x[3, 5:] = -inf
    x[4, [7, 900]] = inf
    x[5, 100:1400] = nan
    x[6] = -inf
    x[6, 1234] = -3.0
    x[7, :] = 0.0
    x[7, ::3] = -0.0
    x[8] = torch.finfo(DTS[dt]).min
    x[9] = torch.finfo(DTS[dt]).min
    x[9, 77] = torch.finfo(DTS[dt]).max
    x[10, 3], x[10, 4] = inf, nan
    for kw in (dict(), dict(temperature=0.0), dict(top_k=4), dict(top_p=0.6), dict(min_p=0.3),
               dict(temperature=0.7, top_k=200, top_p=0.9, min_p=0.01)):
        check_sample(x, u, **kw)


@pytest.mark.parametrize("dt", list(DTS))
def test_sample_strided_rows(dt):
    x, u = logits(dt, 6, 3001, 8)
    check_sample(x[:, 1:2900], u, top_k=20)          # odd offset and row stride
    check_sample(x[::2], u[::2], top_p=0.8)
    check_sample(x[:, ::3], u, top_p=0.8, top_k=100)  # copied first


def test_sample_follows_the_distribution():
    """4096 stratified numbers reproduce the probabilities to one stratum per border."""
    x, _ = logits("f32", 1, 12, 9)
    n = 4096
    u = (torch.arange(n, device=DEV) + 0.5) / n
    got = torch.bincount(ops.sample(x.expand(n, 12), u, temperature=0.8), minlength=12).double() / n
    want = torch.softmax(x[0].double() / float(np.float32(0.8)), 0)
    assert (got - want).abs().max() <= 1.0 / n


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("B", [150, 700])
def test_attention_many_sequences(B, new):
    """More sequences than a block has threads, many of them empty."""
    b = Batch("bf16", [(new if i % 3 else 0, (7 * i) % 90 + new) for i in range(B)], 1, 64, 16, seed=B)
    q, o = attend(b, 2)
    check_attention(b, q, o)


@pytest.mark.parametrize("seqs", [[(1, 20000)], [(1, 20000), (1, 3)], [(40, 30000), (1, 5), (1, 700)]])
def test_attention_one_long_sequence(seqs):
    """One tile cut into more parts than the join looks at in one go."""
    b = Batch("bf16", seqs, 1, 128, 64, seed=18)
    q, o = attend(b, 2)
    check_attention(b, q, o)


@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_attention_decode_long_line(D, dt):
    """Enough keys that CTAs take further pieces of the line when they are done."""
    b = Batch(dt, [(1, 40000), (1, 7), (1, 45000), (0, 0), (1, 300)], 8, D, 64, seed=19)
    q, o = attend(b, 16)
    check_attention(b, q, o)
    for _ in range(5):
        assert torch.equal(attend(b, 16, q=q)[1], o)


def test_attention_decode_wide_table():
    """A table that could name far more keys than there are."""
    b = Batch("bf16", [(1, 100), (1, 2000), (1, 1)], 4, 64, 16, seed=20, stale=float("nan"))
    wide = torch.full((3, 60000), -1, dtype=torch.int32, device=DEV)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide
    q, o = attend(b, 8)
    check_attention(b, q, o)


@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "f16")])
def test_attention_chunks_long_line(D, dt):
    """Chunks whose line is long enough for a second round of pieces, with ragged neighbours."""
    b = Batch(dt, [(300, 9000), (1, 12000), (65, 7000), (0, 0), (2, 2), (130, 20000)], 8, D, 64, seed=21)
    q, o = attend(b, 8)
    check_attention(b, q, o)
    for _ in range(5):
        assert torch.equal(attend(b, 8, q=q)[1], o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("pages", [0, 4])
def test_no_pages_at_all(dt, new, pages):
    """Tables without a column over pools with and without pages: keys are missing, not stored and NaN."""
    b = Batch(dt, [(new, 0), (new, new)], 2, 64, 16, seed=22, spare=4)
    b.kc, b.vc = b.kc[:pages], b.vc[:pages]
    b.table = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    q, o = attend(b, 4)
    assert (o[:new] == 0).all() and o[new:].isnan().all()
    k, v = b.normal(b.N, 2, 64), b.normal(b.N, 2, 64)
    cos, sin = tables(8, 64)
    check_append(b, k, v, q, cos, sin, lambda: ops.paged_append(k, v, b.kc, b.vc, *b.lists(), q=q, cos=cos, sin=sin))


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_over_a_shared_table(dt, new):
    """Sequences that read the same pages: one row of page numbers for all of them."""
    b = Batch(dt, [(new, 150), (new, 150), (new, 90)], 2, 64, 16, seed=23)
    b.table = b.table[:1].expand(3, -1)
    assert b.table.stride(0) == 0
    q, o = attend(b, 4)
    check_attention(b, q, o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 70])
def test_attention_rows_before_the_first_sequence_stay(dt, new):
    b = Batch(dt, [(new, 100), (0, 7), (new, new)], 2, 128, 16, seed=24, rows_behind=5)
    b.cu += 3
    out = torch.full((b.N, 4, 128), 3.0, device=DEV, dtype=b.dt)
    q, o = attend(b, 4, out=out)
    check_attention(b, q, o)
    assert (o[:3] == 3).all() and (o[3 + 2 * new:] == 3).all()


def test_attention_long_line_in_a_graph():
    """A captured call follows the lists as they are when it is replayed."""
    b = Batch("bf16", [(1, 40000), (1, 7), (1, 45000)], 8, 128, 64, seed=25)
    q = b.normal(b.N, 16, 128)
    attend(b, 16, q=q)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        ops.paged_attention(q, b.kc, b.vc, *b.lists(), out=out)
    for lens in ([40000, 7, 45000], [3, 5, 1], [39000, 1, 2000]):
        b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(b, q, out)
        assert torch.equal(out, attend(b, 16, q=q)[1])
