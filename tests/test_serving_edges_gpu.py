"""The serving operators where their arithmetic is at its limits: bounds as in test_serving_gpu.py (h = half
a step of the output type, relative), with what fp16 cannot hold counted:

  attention  fp16 weights P lie at the top of the type's range, the largest so far at least 2^11: one below
             2^-14 is off by at most 2^-25, which is 2^-36 of the row's largest weight.  Decoding splits P
             in two terms, so there only that and 2^-22 (bf16: 2^-17) of the weight itself remain.  fp16
             results below 2^-14 are off by 2^-25.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from autokernel_b200 import ops
from autokernel_b200._lib import device_status

pytestmark = pytest.mark.gpu

DTS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
I32 = torch.int32


def _half(dt):
    return torch.finfo(dt).eps / 2


def one_sequence(k, v, new, length):
    """A cache [1, length, D] (keys, values) in pages of 16 in order, and the lists of `new` tokens."""
    page, D = 16, k.shape[-1]
    P = -(-length // page)
    kc, vc = (torch.zeros(P * page, D, device=DEV, dtype=x.dtype) for x in (k, v))
    kc[:length], vc[:length] = k, v
    lists = (torch.arange(P, dtype=I32, device=DEV)[None], torch.tensor([0, new], dtype=I32, device=DEV),
             torch.tensor([length], dtype=I32, device=DEV))
    return kc.view(P, 1, page, D), vc.view(P, 1, page, D), lists


@pytest.mark.parametrize("gap", [8, 20, 24, 26])
@pytest.mark.parametrize("new", [1, 40, 300])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_weak_keys_beside_leading_ones_without_value(dt, D, new, gap):
    """Every 16th key leads the others by `gap` (log2) and has the value 0: the output is the others' alone."""
    dt, L = DTS[dt], 500
    g = torch.Generator(DEV).manual_seed(gap)
    k = torch.zeros(L, D, device=DEV)
    k[:, 0] = torch.rand(L, device=DEV, generator=g)
    v = 64 + 64 * torch.rand(L, D, device=DEV, generator=g)
    k[::16, 0], v[::16] = gap + 1, 0
    k, v = k.to(dt), v.to(dt)
    q = torch.zeros(new, 2, D, device=DEV, dtype=dt)
    q[..., 0] = 1
    kc, vc, lists = one_sequence(k, v, new, L)
    o = ops.paged_attention(q, kc, vc, *lists, causal=False, sm_scale=math.log(2)).double()
    w = torch.exp2(k[:, 0].double() - (gap + 1))
    w = w / w.max()
    e, A = (w @ v.double()) / w.sum(), (w @ v.double().abs()) / w.sum()
    floor = (v.double().abs().sum(0) / w.sum()) * (2.0 ** -36 if dt == torch.float16 else 0)
    h = _half(dt)
    hp = h if new > 1 else 2.0 ** -22 if dt == torch.float16 else 2.0 ** -17
    d = (D + 8) * 2.0 ** -24 * (gap + 1) + 2.0 ** -20
    tol = torch.clamp(h * e, min=2.0 ** -25 if dt == torch.float16 else 0) + (hp + 2 * d + (L + 8) * 2.0 ** -23) * A + floor
    err = (o - e).abs()
    assert (err <= tol).all(), (float((err / e).max()), float((tol / e).min()))


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("mag", [1e3, 5e3, 2e4, 5e4])
@pytest.mark.parametrize("new", [1, 300])
def test_scores_whose_steps_are_large(dt, mag, new):
    """Scores up to 1e10, whose fp32 steps are 1 and more: which key wins is a matter of rounding, but a row stays a
    mean of the values, or is NaN where its largest score (scaled, log2) is beyond 2^27 (fp16) or 2^31
    (bf16): no 16-bit weights reach from there.  fp32 has no such border."""
    dt, L, D = DTS[dt], 310, 64
    g = torch.Generator(DEV).manual_seed(2)
    k, q = ((torch.randn(n, D, device=DEV, generator=g) * mag).clamp(-6e4, 6e4).to(dt) for n in (L, new * 2))
    v = torch.randn(L, D, device=DEV, generator=g).to(dt)
    kc, vc, lists = one_sequence(k, v, new, L)
    o = ops.paged_attention(q.view(new, 2, D), kc, vc, *lists).double()
    score = (q.double() @ k.double().T).view(new, 2, L) * D ** -0.5 / math.log(2)
    hidden = torch.arange(L, device=DEV) > torch.arange(L - new, L, device=DEV)[:, None, None]
    top = score.masked_fill(hidden, -math.inf).amax(-1).abs()
    limit = {torch.float16: 2.0 ** 27, torch.bfloat16: 2.0 ** 31, torch.float32: math.inf}[dt]
    near = (D + 8) * 2.0 ** -24 * (q.double().abs() @ k.double().abs().T).amax(-1).view(new, 2) * D ** -0.5 / math.log(2)
    inside, beyond = top + near < limit, top - near > limit
    assert o[inside].isfinite().all() and o[beyond].isnan().all()
    if mag == 1e3:
        assert inside.all()
    # weights sum to 1 but for their rounding (h) and that of the sums
    most = v.double().abs().amax(0) * (1 + 2 * _half(dt) + 2 * (L + 8) * 2.0 ** -23)
    assert ((o.abs() <= most) | o.isnan()).all()
    assert device_status() == 0


@pytest.mark.parametrize("dt,D", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("seqs,heads,kv", [([(1, 3000), (3, 900)] + 6 * [(1, 1500)], 600, 300),
                                           ([(1, 300 + 119 * i) for i in range(64)], 32, 8)])
def test_decoding_gives_the_same_bits_every_time(seqs, heads, kv, D, dt):
    """CTAs take pieces of a long line as they become free: which one took which does not show in the result."""
    seqs = seqs + [(0, 0)] * (sum(s[0] for s in seqs) - len(seqs))
    g = torch.Generator(DEV).manual_seed(3)
    page = 16
    used = [-(-s[1] // page) for s in seqs]
    table = torch.full((len(seqs), max(used)), -1, dtype=I32)
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(sum(used[:b]), sum(used[:b]) + n)
    cu = torch.tensor([sum(s[0] for s in seqs[:i]) for i in range(len(seqs) + 1)], dtype=I32, device=DEV)
    lists = (table.to(DEV), cu, torch.tensor([s[1] for s in seqs], dtype=I32, device=DEV))
    kc, vc = (torch.randn(sum(used), kv, page, D, device=DEV, dtype=DTS[dt], generator=g) for _ in range(2))
    q = torch.randn(int(cu[-1]), heads, D, device=DEV, dtype=DTS[dt], generator=g)
    first = ops.paged_attention(q, kc, vc, *lists)
    for _ in range(20):
        assert torch.equal(ops.paged_attention(q, kc, vc, *lists), first)


def packed(seqs, heads, kv_heads, D, dt, page=16, seed=0):
    """(q, k_cache, v_cache, lists) of sequences (new tokens, keys) whose pages lie in order, and their keys'
    places in the caches."""
    g = torch.Generator(DEV).manual_seed(seed)
    new, lens = [s[0] for s in seqs], [s[1] for s in seqs]
    used = [-(-x // page) for x in lens]
    first = [sum(used[:i]) for i in range(len(used))]
    table = torch.full((len(seqs), max(used + [1])), -1, dtype=I32)
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(first[b], first[b] + n)
    kc, vc = (torch.randn(sum(used), kv_heads, page, D, device=DEV, dtype=dt, generator=g) for _ in range(2))
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=I32, device=DEV)
    q = torch.randn(sum(new), heads, D, device=DEV, dtype=dt, generator=g)
    return q, kc, vc, (table.to(DEV), cu, torch.tensor(lens, dtype=I32, device=DEV)), first


def near_64_bits(q, kc, vc, lists, seqs, first, o, rows, heads, page=16):
    """Rows `rows` (sequence, token) of some heads against the formula in 64 bits, within the bound of
    test_serving_gpu.py."""
    G, D, h = q.shape[1] // kc.shape[1], q.shape[2], _half(q.dtype)
    cu = lists[1].tolist()
    for b, i in rows:
        new, length = seqs[b]
        vis = length - new + i + 1
        for head in heads:
            at = torch.arange(vis, device=DEV)
            k, v = (c[first[b] + at // page, head // G, at % page].double() for c in (kc, vc))
            x = q[cu[b] + i, head].double()
            w = torch.softmax(k @ x * D ** -0.5, 0)
            e, A = w @ v, w @ v.abs()
            d = (D + 8) * 2.0 ** -24 * (k.abs() @ x.abs()).max() * D ** -0.5 + 2.0 ** -20
            tol = h * e.abs() + (h + 2 * d + (vis + 8) * 2.0 ** -23) * A
            err = (o[cu[b] + i, head].double() - e).abs()
            assert (err <= tol).all(), (b, i, head, float((err - tol).max()))


HIDDEN = [  # sequences, heads, kv heads, D: chunks cut into parts and whole in a piece, then decoding tiles
    ([(256, 100000), (1, 50)], 1, 1, 64), ([(200, 200000)], 1, 1, 128), ([(64, 30000), (3, 77)], 4, 1, 128),
    ([(250, 6000)], 300, 300, 64), ([(40, 3000), (60, 900)], 300, 300, 128),
    ([(5, 100000), (1, 9)] + 6 * [(0, 0)], 2, 2, 64), ([(3, 3000), (2, 400)] + 6 * [(0, 0)], 600, 300, 128),
    ([(4, 20000)] + 6 * [(0, 0)], 64, 16, 64)]


@pytest.mark.parametrize("dt,value", [("f16", float("inf")), ("bf16", float("nan"))])
@pytest.mark.parametrize("case", range(len(HIDDEN)))
def test_hidden_infinities_under_long_contexts(case, dt, value):
    """The value of a chunk's last token is not finite: the tokens before it, which share its tile and see long
    contexts, are as without it; so are the other sequences, and no wait runs out."""
    seqs, heads, kv, D = HIDDEN[case]
    q, kc, vc, lists, first = packed(seqs, heads, kv, D, DTS[dt], seed=case)
    clean = ops.paged_attention(q, kc, vc, *lists)
    new, length = seqs[0]
    vc[first[0] + (length - 1) // 16, :, (length - 1) % 16] = value
    o = ops.paged_attention(q, kc, vc, *lists)
    again = ops.paged_attention(q, kc, vc, *lists)
    torch.cuda.synchronize()
    assert device_status() == 0
    rest = torch.arange(o.shape[0], device=DEV) != new - 1
    assert o[rest].isfinite().all() and not o[new - 1].isfinite().any()
    assert torch.equal(o[rest], again[rest])
    # the clean call rounds its weights to 16 bits, so it differs; rows of other sequences do not
    assert torch.equal(o[new:], clean[new:])
    some = [(0, i) for i in sorted({0, new // 2, new - 2})]
    if len(seqs) > 1 and seqs[1][0]:
        some.append((1, seqs[1][0] - 1))
    near_64_bits(q, kc, vc, lists, seqs, first, o, some, sorted({0, heads // 2, heads - 1}))


def _model(dtype=torch.float16, heads=4, dim=256):
    from autokernel_b200.llama import LlamaB200, LlamaConfig
    c = LlamaConfig(vocab_size=512, dim=dim, n_layers=2, n_heads=heads, n_kv_heads=2, hidden_dim=512)
    return LlamaB200(c, LlamaB200.random_weights(c, DEV, dtype=dtype, seed=3, std=0.05))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 70, 3]])
def test_a_token_outside_of_the_vocabulary_stays_in_its_sequence(dtype, counts):
    m = _model(dtype)
    cache = m.new_cache(40, 16)
    seqs = [cache.add() for _ in counts]
    g = torch.Generator().manual_seed(1)

    def step(counts, bad):
        batch = cache.extend(seqs, counts)
        tokens = torch.randint(0, 512, (sum(counts),), generator=g)
        out = []
        for at in (None, bad):  # twice over the same keys: they are written again
            t = tokens.clone()
            if at is not None:
                t[at] = [-1, 512, 2 ** 40][at % 3]
            out.append(m.extend(t.to(DEV), batch, cache))
        return out

    step([20, 33, 5], None)
    good, bad = step(counts, counts[0])  # the second sequence's first token
    assert torch.equal(good[[0, 2]], bad[[0, 2]]) and good.isfinite().all() and bad[1].isnan().all()
    good, bad = step([1, 1, 1], None)
    assert good[[0, 2]].isfinite().all() and good[1].isnan().all()
    assert ops.sample(good, torch.rand(3, device=DEV)).tolist()[1] == -1
    assert device_status() == 0


def test_generate_with_settings_of_each_prompt():
    m = _model()
    prompts = [[1, 2, 3], [7] * 70, [5]]
    greedy = m.generate(prompts, 6, temperature=0.0)
    got = m.generate(prompts, 6, temperature=[0.0, 1.0, 0.0], top_k=torch.tensor([0, 50, 0]), top_p=[1.0, 0.9, 1.0],
                     generator=torch.Generator(DEV).manual_seed(1))
    assert got[0] == greedy[0] and got[2] == greedy[2] and len(got[1]) == 6


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("vocab", [700, 40000])
def test_infinite_temperature_among_dead_logits(dt, vocab):
    """Every alive entry weighs the same; NaN and -inf, and what top-k left out, weigh nothing."""
    from oracle import serve_f64
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.randn(12, vocab, device=DEV, generator=g).to(DTS[dt])
    x[::2, ::3] = -math.inf
    x[::3, 1::4] = math.nan
    x[4:6] = torch.where(x[4:6].isfinite(), 1.0, x[4:6])
    u = torch.rand(12, device=DEV, generator=g)
    for kw in (dict(top_p=0.5), dict(top_p=0.001), dict(top_p=0.999), dict(top_k=vocab // 2, top_p=0.3), dict(min_p=0.5), dict()):
        got = ops.sample(x, u, temperature=math.inf, **kw).tolist()
        kw = {k: float(np.float32(v)) if k != "top_k" else v for k, v in kw.items()}
        assert got == [serve_f64.sample_row(x[r].double().cpu().numpy(), u[r].item(), math.inf, **kw) for r in range(12)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,D,seqs", [
    (64, 8, 128, [(1, 20 + 37 * i) for i in range(40)]),                     # 8 rows a sequence, many pairs
    (64, 8, 64, [(1, 700)] * 3),                                             # 8 rows, few pairs
    (32, 2, 128, [(1, 333), (1, 64), (1, 1)]),                               # 16
    (40, 1, 64, [(1, 500), (1, 3)]),                                         # 40
    (32, 8, 128, [(1, 50 + i) for i in range(50)] + [(2, 99)]),              # one of two tokens
    (16, 8, 64, [(0, 0)] * 30 + [(61, 400), (1, 77)] + [(0, 0)] * 30),       # slots, one of them a chunk
    (8, 8, 128, [(5, 90), (9, 9), (4, 250)] + [(1, 30 + i) for i in range(40)])])
def test_groups_and_batches_of_all_widths(heads, kv, D, seqs, dt):
    """Calls on both sides of the rule that chooses a kernel, each row against the formula."""
    q, kc, vc, lists, first = packed(seqs, heads, kv, D, DTS[dt], seed=heads + D)
    o = ops.paged_attention(q, kc, vc, *lists)
    rows = [(b, i) for b, (new, _) in enumerate(seqs) for i in sorted({0, new // 2, new - 1}) if new]
    near_64_bits(q, kc, vc, lists, seqs, first, o, rows, sorted({0, heads // 2, heads - 1}))


@pytest.mark.parametrize("heads,kv,n", [(32, 2, 1), (8, 8, 3)])
def test_a_call_whose_lists_change_under_a_graph(heads, kv, n):
    """64 slots, captured once: the lists may spread the tokens over the sequences in any way."""
    B, D, page = 64, 128, 16
    g = torch.Generator(DEV).manual_seed(9)
    q = torch.randn(B * n, heads, D, device=DEV, generator=g).half()
    kc, vc = (torch.randn(B * 4, kv, page, D, device=DEV, generator=g).half() for _ in range(2))
    table = torch.arange(B * 4, device=DEV, dtype=I32).view(B, 4)
    cu, lens = torch.zeros(B + 1, dtype=I32, device=DEV), torch.zeros(B, dtype=I32, device=DEV)
    out = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, cu, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, kc, vc, table, cu, lens, out=out)
    for seqs in ([(n, 20 + b % 40) for b in range(B)], [(0, 0)] * 60 + [(40, 64), (0, 9), (23, 30), (1, 1)], [(0, 64)] * B):
        cu.copy_(torch.tensor([sum(s[0] for s in seqs[:i]) for i in range(B + 1)], dtype=I32))
        lens.copy_(torch.tensor([s[1] for s in seqs], dtype=I32))
        out.fill_(7.0)
        graph.replay()
        rows = [(b, s[0] - 1) for b, s in enumerate(seqs) if s[0]]
        near_64_bits(q, kc, vc, (table, cu, lens), seqs, [4 * b for b in range(B)], out, rows, [0, heads - 1])
        assert (out[int(cu[-1]):] == 7).all()


@pytest.mark.parametrize("dt,D", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("seqs", [
    [(1, 100 + b) for b in range(20)] + [(1, 26000), (3, 25000), (1, 27000)] + [(1, 1 + b) for b in range(15)] + [(0, 50), (0, 0)],
    [(1, 90 + b % 40) for b in range(600)] + [(1, 400), (2, 700)]])
def test_decoding_in_rounds_of_pieces(seqs, D, dt):
    """Lines long enough for rounds, with tiles that several pieces share and pieces that hold many tiles; then
    other lists under the same captured call, a short line among them."""
    q, kc, vc, lists, first = packed(seqs, 16, 8, D, DTS[dt], seed=D)
    o = ops.paged_attention(q, kc, vc, *lists)
    live = [b for b, s in enumerate(seqs) if s[0]]
    some = sorted({*live[:2], *live[len(live) // 2 - 2:len(live) // 2 + 4], *live[-3:]})
    near_64_bits(q, kc, vc, lists, seqs, first, o, [(b, seqs[b][0] - 1) for b in some], [0, 7, 15])
    out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, kc, vc, *lists, out=out)
    graph.replay()
    assert torch.equal(out, o)
    short = [(n, min(x, 40 + b % 30)) for b, (n, x) in enumerate(seqs)]
    lists[2].copy_(torch.tensor([s[1] for s in short], dtype=I32))
    graph.replay()
    near_64_bits(q, kc, vc, lists, short, first, out, [(b, short[b][0] - 1) for b in some], [0, 15])


@pytest.mark.parametrize("dt", list(DTS))
@pytest.mark.parametrize("heads,kv,D,page", [(8, 2, 128, 16), (3, 1, 80, 5), (2, 2, 6, 3), (32, 32, 64, 64)])
def test_append_rotation_element_by_element(dt, heads, kv, D, page):
    """Each rotated element within h |e| (2^-25 where fp16 is subnormal) + 3 * 2^-24 of what its own sum adds up:
    two fp32 products, their sum, one rounding.  Sizes from 1e-3 to 1e3 within a vector."""
    from oracle import serve_f64
    dt, seqs = DTS[dt], [(7, 23), (1, 90), (40, 64), (0, 3), (130, 131)]
    g = torch.Generator(DEV).manual_seed(D)
    q, kc, vc, lists, first = packed(seqs, heads, kv, D, dt, page, seed=D)
    k = torch.randn(q.shape[0], kv, D, device=DEV, generator=g)
    spread = 10 ** (6 * torch.rand(D, device=DEV, generator=g) - 3)
    q, k = (q * spread).to(dt), (k * spread).to(dt)
    angle = torch.rand(140, D // 2, device=DEV, generator=g, dtype=torch.float64) * 6.3
    cos, sin = angle.cos().float(), angle.sin().float()
    out = ops.paged_append(k, k, kc, vc, *lists, q=q, cos=cos, sin=sin)
    h, floor = _half(dt), 2.0 ** -25 if dt == torch.float16 else 0
    cu, n64 = lists[1].tolist(), lambda t: t.double().cpu().numpy()  # noqa: E731
    for b, (new, length) in enumerate(seqs):
        at = np.arange(length - new, length)
        c, s = n64(cos)[at][:, None], n64(sin)[at][:, None]
        stored = kc[first[b] + torch.tensor(at // page, device=DEV), :, torch.tensor(at % page, device=DEV)]
        for x, y in ((q, out[cu[b]:cu[b + 1]]), (k, stored)):
            x = n64(x[cu[b]:cu[b + 1]])
            e, size = serve_f64.rotate(x, c, s), serve_f64.rotate_size(x, c, s)
            assert (np.abs(n64(y) - e) <= np.maximum(h * np.abs(e), floor) + 3 * 2.0 ** -24 * size).all()


def test_calls_on_several_streams_at_once():
    """Decoding in rounds, decoding of one, chunks and sampling side by side: each as if it were alone."""
    def attention(seqs, heads, kv, D):
        q, kc, vc, lists, _ = packed(seqs, heads, kv, D, torch.float16, seed=len(seqs))
        return lambda: ops.paged_attention(q, kc, vc, *lists)

    g = torch.Generator(DEV).manual_seed(1)
    x, u = torch.randn(40, 30000, device=DEV, generator=g), torch.rand(40, device=DEV, generator=g)
    calls = [attention([(1, 100 + 97 * i) for i in range(48)], 32, 8, 128), attention([(1, 3000)], 8, 8, 64),
             attention([(130, 2000), (1, 700), (33, 33)], 8, 2, 128), lambda: ops.sample(x, u, 0.9, 0, 0.8)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(20):
        got = []
        for i, (f, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got.append([f() for _ in range(1 + (turn + i) % 3)])
        torch.cuda.synchronize()
        for w, results in zip(want, got):
            assert all(torch.equal(w, r) for r in results)
    assert device_status() == 0


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("new", [1, 40, 300])
@pytest.mark.parametrize("far", ["first", "last", "most", "all but one", "all"])
def test_scores_far_below_the_others(dt, new, far):
    """Keys whose scores are -3e8 (fp16) or -1e10: beside others they weigh nothing, wherever they lie; a row that
    sees no others is NaN in 16 bits (no 16-bit weights reach from there), a mean of their values in fp32."""
    dt, L, D = DTS[dt], 3000, 64
    g = torch.Generator(DEV).manual_seed(6)
    k, v = (torch.randn(L, D, device=DEV, generator=g) for _ in range(2))
    q = torch.randn(new, 2, D, device=DEV, generator=g)
    at = torch.zeros(L, dtype=torch.bool, device=DEV)
    if far == "first":
        at[:1700] = True
    elif far == "last":
        at[1300:] = True
    else:
        at[:] = True
        at[{"most": torch.arange(5, L, 97), "all but one": torch.tensor([1234]), "all": torch.arange(0)}[far]] = False
    big = 3e4 if dt == torch.float16 else 1e5
    k[:, 0], q[..., 0] = torch.where(at, -big / 3 if dt == torch.float16 else -big, 0.0), big
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    kc, vc, lists = one_sequence(k, v, new, L)
    o = ops.paged_attention(q, kc, vc, *lists, causal=False, sm_scale=1.0).double()
    if far == "all":
        assert o.isfinite().all() if dt == torch.float32 else o.isnan().all()
        return
    s = torch.where(at, -math.inf, q.double() @ k.double().T)
    w = torch.softmax(s, -1)
    e, A, h = w @ v.double(), w @ v.double().abs(), _half(dt)
    d = (D + 8) * 2.0 ** -24 * (q.double().abs() @ torch.where(at[:, None], 0.0, k.double()).abs().T).amax(-1, keepdim=True)
    floor = (2.0 ** -36 if dt == torch.float16 else 0) * v.double().abs().sum(0)
    tol = torch.clamp(h * e.abs(), min=2.0 ** -25 if dt == torch.float16 else 0) + (h + 2 * (d + 2.0 ** -20) + (L + 8) * 2.0 ** -23) * A + floor
    assert ((o - e).abs() <= tol).all()
