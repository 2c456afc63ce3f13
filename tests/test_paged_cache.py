"""PagedCache's bookkeeping (on the CPU), the dispatcher schemas of the serving operators, and LlamaB200
answering over the cache on a GPU: every step's logits against the float64 model of the whole
sequence."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import autokernel_b200.torch_ops  # noqa: F401
from autokernel_b200 import AkError
from autokernel_b200.paged import PagedCache
from oracle import llama_f64
from parity import check

AK = torch.ops.autokernel_b200


def _cache(pages=10, page=4):
    return PagedCache(2, 3, 8, pages, page, torch.float32, "cpu")


def test_pages_are_handed_out_and_given_back():
    c = _cache()
    a, b = c.add(), c.add()
    x = c.extend([a, b], [5, 4])
    assert x.cu_q.tolist() == [0, 5, 9] and x.kv_lens.tolist() == [5, 4]
    assert x.n_tokens == 9 and x.max_len == 5 and x.page_table.shape == (2, 2)
    assert x.page_table[1, 1] == -1 and c.free_pages == 7
    y = c.extend([b], [1])
    assert y.kv_lens.tolist() == [5] and y.page_table.tolist() == [c.pages(b)] and len(c.pages(b)) == 2
    assert not set(c.pages(a)) & set(c.pages(b))
    assert c.length(a) == 5 and c.length(b) == 5
    c.release(a)
    assert c.free_pages == 8
    with pytest.raises(KeyError):
        c.length(a)
    c.release(b)
    assert c.free_pages == 10
    assert {t.shape for t in c.k + c.v} == {torch.Size([10, 3, 4, 8])}


def test_a_full_cache_refuses_and_stays_as_it_was():
    c = _cache(pages=3)
    a, b = c.add(), c.add()
    c.extend([a], [8])
    with pytest.raises(AkError, match="full"):
        c.extend([a, b], [1, 5])
    assert c.length(a) == 8 and c.length(b) == 0 and c.free_pages == 1
    c.extend([a], [4])
    assert c.free_pages == 0


def test_extend_refusals():
    c = _cache()
    a = c.add()
    for seqs, counts in (([], []), ([a], [1, 2]), ([a, a], [1, 1]), ([a], [0])):
        with pytest.raises(ValueError):
            c.extend(seqs, counts)
    with pytest.raises(KeyError):
        c.extend([99], [1])
    with pytest.raises(ValueError):
        PagedCache(1, 1, 0, 4)


def test_fake_shapes():
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    cache = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    lists = [torch.zeros(*s, dtype=torch.int32) for s in ((2, 3), (3,), (2,))]
    cos = torch.zeros(99, 32)
    with FakeTensorMode() as mode:
        f = mode.from_tensor
        fl = [f(t) for t in lists]
        assert AK.paged_append(f(k), f(k), f(cache), f(cache), *fl, f(q), f(cos), f(cos)).shape == q.shape
        o = AK.paged_attention(f(q), f(cache), f(cache), *fl)
        assert o.shape == q.shape and o.dtype == q.dtype
        t = AK.sample(f(torch.zeros(7, 100)), f(torch.zeros(7)), 0.5, 3)
        assert t.shape == (7,) and t.dtype == torch.int64


def _model(dtype, n_kv=2, fuse=None, heads=4, dim=512):
    from autokernel_b200.llama import LlamaB200, LlamaConfig
    c = LlamaConfig(vocab_size=512, dim=dim, n_layers=2, n_heads=heads, n_kv_heads=n_kv, hidden_dim=1024)
    w = LlamaB200.random_weights(c, "cuda", dtype=dtype, seed=3, std=0.05)
    return LlamaB200(c, w, fuse_norms=fuse)


def _logits64(m, tokens):
    sd = {k: v.double().cpu().numpy() for k, v in m.w.items()}
    return llama_f64.forward(sd, torch.tensor([tokens]).numpy(), m.cfg.n_heads, m.cfg.n_kv_heads)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fuse,heads,scale_tol", [
    (torch.float16, None, 4, 2.0), (torch.bfloat16, None, 4, 10.0), (torch.float16, False, 4, 2.0),
    (torch.float16, None, 8, 2.0), (torch.float16, None, 16, 2.0), (torch.float32, None, 4, 2.0)])
def test_steps_match_the_whole_sequence(dtype, fuse, heads, scale_tol):
    """Prompts of several lengths, a second chunk, then single tokens, sequences leaving and joining: each
    step's logits are those of the float64 model over the sequence so far (the tolerances of the
    whole forward's test: the arithmetic between the layers is the same)."""
    m = _model(dtype, fuse=fuse, heads=heads)
    cache = m.new_cache(40, 16)
    g = torch.Generator().manual_seed(1)

    def some(n):
        return torch.randint(0, 512, (n,), generator=g).tolist()

    text = {cache.add(): [] for _ in range(3)}
    a, b, c = text
    d = cache.add()
    text[d] = []
    for chunk in ({a: 150, b: 3, c: 17}, {a: 40, c: 1}, {a: 1, b: 1, c: 1}, {b: 1, c: 1, d: 33}, {c: 1, b: 1},
                  {d: 2, a: 1}):
        new = {s: some(n) for s, n in chunk.items()}
        batch = cache.extend(list(new), [len(t) for t in new.values()])
        logits = m.extend(torch.tensor([t for x in new.values() for t in x], device="cuda"), batch, cache)
        for row, (s, t) in enumerate(new.items()):
            text[s] += t
            e = _logits64(m, text[s])[-1]
            check(logits[row], e, "matmul", "cached llama", scale_tol=scale_tol)
    assert cache.length(a) == len(text[a])


@pytest.mark.gpu
def test_generate():
    m = _model(torch.float16)
    prompts = [[1, 2, 3], [7] * 70, [5]]
    # the likeliest token of every step, from the whole forward
    got = m.generate(prompts, 6, temperature=0.0)
    for p, t in zip(prompts, got):
        assert len(t) == 6
        e = _logits64(m, p + t)
        for i, x in enumerate(t):
            row = e[len(p) - 1 + i]
            assert row[x] >= row.max() - 0.04  # two logits this close may change places in 16 bits
    # the same numbers, the same tokens; other ones, others; and all pages come back
    cache = m.new_cache(12, 16)
    draw = lambda seed: m.generate(prompts, 9, 1.0, 50, 0.95, 0.01, cache=cache,  # noqa: E731
                                   generator=torch.Generator("cuda").manual_seed(seed))
    first = draw(1)
    assert first == draw(1) and first != draw(2)
    assert cache.free_pages == 12
    # a sequence ends with the stop token
    stop = first[0][4]
    ended = m.generate(prompts, 9, 1.0, 50, 0.95, 0.01, stop=stop, cache=cache,
                       generator=torch.Generator("cuda").manual_seed(1))
    assert ended[0] == first[0][:first[0].index(stop) + 1]
    assert cache.free_pages == 12
    with pytest.raises(AkError):
        m.generate([[1] * 300], 1, cache=cache)
    assert cache.free_pages == 12
    assert m.generate([[1]], 0) == [[]]
    for bad in ([], [[]], [[1], []]):
        with pytest.raises(ValueError):
            m.generate(bad, 3)


@pytest.mark.gpu
def test_generate_refuses_what_it_cannot_embed():
    m = _model(torch.float16)
    vocab = m.w["tok_embeddings.weight"].shape[0]
    for bad in ([[vocab]], [[1, 2], [-1]]):
        with pytest.raises(ValueError, match="tokens"):
            m.generate(bad, 2)
    m.w["output.weight"] = torch.full_like(m.w["output.weight"], float("nan"))
    cache = m.new_cache(4, 16)
    for stop in (None, 0):
        with pytest.raises(AkError, match="draw"):
            m.generate([[1, 2], [3]], 3, stop=stop, cache=cache)
        assert cache.free_pages == 4


@pytest.mark.gpu
def test_decoding_step_in_a_graph():
    """A captured decoding step (append, attention, sampling) replayed with other lists, tokens and
    numbers gives what eager calls give; a padded row of the batch stays as it was."""
    from autokernel_b200 import ops
    g = torch.Generator("cuda").manual_seed(2)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g).half()

    B, H, Hkv, D, page = 4, 8, 2, 128, 16
    kc, vc = normal(30, Hkv, page, D), normal(30, Hkv, page, D)
    table = torch.randperm(30, device="cuda", generator=g)[:28].view(4, 7).int()
    cu = torch.tensor([0, 1, 2, 3, 3], dtype=torch.int32, device="cuda")  # the last row is padding
    lens = torch.tensor([5, 100, 33, 0], dtype=torch.int32, device="cuda")
    q, k, v, logits, u = normal(B, H, D), normal(B, Hkv, D), normal(B, Hkv, D), normal(B, 999), torch.rand(B, device="cuda")
    cos, sin = torch.rand(200, D // 2, device="cuda"), torch.rand(200, D // 2, device="cuda")
    out, rot = torch.full_like(q, 9.0), torch.full_like(q, 9.0)

    def step():
        ops.paged_append(k, v, kc, vc, table, cu, lens, q=q, cos=cos, sin=sin, q_out=rot)
        ops.paged_attention(rot, kc, vc, table, cu, lens, out=out)
        return ops.sample(logits, u, 0.8, 40, 0.9)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = step()
    for new in ([6, 101, 34, 0], [7, 110, 48, 0], [1, 64, 112, 0]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        for t in (q, k, v, logits):
            t.copy_(normal(*t.shape))
        u.uniform_(generator=g)
        keep = kc.clone(), vc.clone()
        out.fill_(9.0)
        rot.fill_(9.0)
        graph.replay()
        got = [t.clone() for t in (tokens, out, rot, kc, vc)]
        kc.copy_(keep[0])
        vc.copy_(keep[1])
        out.fill_(9.0)
        rot.fill_(9.0)
        want = [step(), out, rot, kc, vc]
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert (got[1][3] == 9).all() and (got[2][3] == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 200])
def test_two_graphs_on_two_streams(tokens):
    """Two captured calls replayed at once do not share their workspaces."""
    from autokernel_b200 import ops
    g = torch.Generator("cuda").manual_seed(4)
    H, Hkv, D, page = 8, 2, 128, 16
    made = []
    for _ in range(2):
        kc, vc = (torch.randn(150, Hkv, page, D, device="cuda", generator=g).half() for _ in range(2))
        table = torch.randperm(150, device="cuda", generator=g).view(3, 50).int()
        n = [1, 1, 1] if tokens == 3 else [tokens - 2, 1, 1]
        cu = torch.tensor([0, n[0], n[0] + 1, n[0] + 2], dtype=torch.int32, device="cuda")
        lens = torch.tensor([800, 500, 333], dtype=torch.int32, device="cuda")
        q = torch.randn(tokens, H, D, device="cuda", generator=g).half()
        args = (q, kc, vc, table, cu, lens)
        want = ops.paged_attention(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention(*args)
        made.append((graph, out, want, args))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(30):
        for (graph, _, _, _), st in zip(made, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in made:
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_registered_serving_ops():
    from autokernel_b200 import ops
    g = torch.Generator("cuda").manual_seed(3)
    q, k = (torch.randn(2, h, 64, device="cuda", generator=g).half() for h in (4, 2))
    kc, vc = (torch.randn(5, 2, 16, 64, device="cuda", generator=g).half() for _ in range(2))
    lists = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 1], [2, 4]], [0, 1, 2], [20, 7])]
    cos, sin = torch.rand(99, 32, device="cuda"), torch.rand(99, 32, device="cuda")
    kc2, vc2 = kc.clone(), vc.clone()
    r = AK.paged_append(k, k, kc, vc, *lists, q, cos, sin)
    assert torch.equal(r, ops.paged_append(k, k, kc2, vc2, *lists, q=q, cos=cos, sin=sin))
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    assert torch.equal(AK.paged_attention(r, kc, vc, *lists), ops.paged_attention(r, kc, vc, *lists))
    x, u = torch.randn(6, 300, device="cuda", generator=g), torch.rand(6, device="cuda")
    assert torch.equal(AK.sample(x, u, 0.7, 20, 0.9, 0.0), ops.sample(x, u, 0.7, 20, 0.9, 0.0))
    for op, args in ((AK.paged_append, (k, k, kc, vc, *lists, q, cos, sin)),
                     (AK.paged_attention, (q, kc, vc, *lists)), (AK.sample, (x, u))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def test_a_sequence_can_be_shortened():
    """What extend() counted and nobody ran is taken back, pages included."""
    c = _cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [6, 3])
    first = c.pages(a)
    c.extend([a], [11])
    assert c.free_pages == 4 and len(c.pages(a)) == 5
    c.truncate(a, 6)
    assert c.length(a) == 6 and c.pages(a) == first and c.free_pages == 7
    c.truncate(a, 4)
    assert c.pages(a) == first[:1] and c.free_pages == 8
    x = c.extend([a], [1])
    assert x.kv_lens.tolist() == [5] and x.page_table[0, 0] == first[0]
    assert not set(c.pages(a)) & set(c.pages(b))
    c.truncate(a, 5)
    c.truncate(a, 0)
    assert c.length(a) == 0 and c.pages(a) == [] and c.free_pages == 9
    for n in (-1, 1):
        with pytest.raises(ValueError, match="truncate"):
            c.truncate(a, n)
    with pytest.raises(KeyError):
        c.truncate(77, 0)


def test_fake_shapes_of_the_second_forms():
    k, cache = torch.zeros(5, 2, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    lists = [torch.zeros(*s, dtype=torch.int32) for s in ((2, 3), (3,), (2,))]
    with FakeTensorMode() as mode:
        f = mode.from_tensor
        assert AK.paged_append_kv(f(k), f(k), f(cache), f(cache), *[f(t) for t in lists]) is None
        row = f(torch.zeros(7))
        t = AK.sample_rows(f(torch.zeros(7, 100)), row, row, f(torch.zeros(7, dtype=torch.int32)), row, row)
        assert t.shape == (7,) and t.dtype == torch.int64


@pytest.mark.gpu
def test_registered_second_forms():
    from autokernel_b200 import ops
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(2, 2, 64, device="cuda", generator=g).half() for _ in range(2))
    lists = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 1], [2, 4]], [0, 1, 2], [20, 7])]
    cos, sin = torch.rand(99, 32, device="cuda"), torch.rand(99, 32, device="cuda")
    for tables in ((), (cos, sin)):
        kc, vc = (torch.randn(5, 2, 16, 64, device="cuda", generator=g).half() for _ in range(2))
        kc2, vc2 = kc.clone(), vc.clone()
        AK.paged_append_kv(k, v, kc, vc, *lists, *tables)
        ops.paged_append(k, v, kc2, vc2, *lists, **dict(zip(("cos", "sin"), tables)))
        assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
        torch.library.opcheck(AK.paged_append_kv, (k, v, kc, vc, *lists, *tables),
                              test_utils=("test_schema", "test_faketensor"))
    x, u = torch.randn(6, 300, device="cuda", generator=g), torch.rand(6, device="cuda")
    t, p, m = torch.rand(6, device="cuda"), torch.rand(6, device="cuda"), torch.rand(6, device="cuda") * 0.1
    n = torch.tensor([0, 1, 5, 50, 0, 299], dtype=torch.int32, device="cuda")
    assert torch.equal(AK.sample_rows(x, u, t, n, p, m), ops.sample(x, u, t, n, p, m))
    torch.library.opcheck(AK.sample_rows, (x, u, t, n, p, m), test_utils=("test_schema", "test_faketensor"))
