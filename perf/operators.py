"""Cases that measure the operators a LLaMA answers with: appending to a paged key/value cache,
attention over that cache and sampling the next token.

Each operator has a plain form of elementary torch operations (32-bit, or 64-bit where sums decide
between neighbouring values) and the framework's own (``own``).  ``exact`` restates the definition
in 64 bits.

Layout shared by the cache operators: N tokens of B sequences are packed one after another, tokens
cu_q[b]..cu_q[b+1] belong to sequence b; kv_lens[b] counts its keys with the new ones; position p
of sequence b lies in slot p % S of page page_table[b, p // S] of caches [P, Hkv, S, D].
"""
import random

import torch

own = False

_DTYPE = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_SIZE = {"bfloat16": 2, "float16": 2, "float32": 4}
_MAX_POSITIONS = 8192  # rows of the rotation tables


# ------------------------------------------------------------------------------------ cases

def _append(name, dtype, seqs, new, old, heads, kv_heads, head_dim, page, fused):
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "new_lo": new[0],
            "new_hi": new[1], "old_lo": old[0], "old_hi": old[1], "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "fused": fused}


def _attend(name, dtype, seqs, new, old, heads, kv_heads, head_dim, page, causal=True):
    return {"name": name, "op": "attention", "dtype": dtype, "seqs": seqs, "new_lo": new[0],
            "new_hi": new[1], "old_lo": old[0], "old_hi": old[1], "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "causal": causal}


def _sample(name, dtype, rows, vocab, temperature, top_k, top_p, min_p, mixed=False):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "mixed": mixed}


def listed():
    return [
        # one user, one token: the LLaMA-7B layer (32 heads of 128) a chat decodes with
        _append("append_one", "bfloat16", 1, (1, 1), (1999, 1999), 32, 32, 128, 16, False),
        # a full serving batch of single tokens, grouped heads, views of one fused projection
        _append("append_batch", "float16", 200, (1, 1), (17, 4000), 32, 8, 128, 16, True),
        # a step that prefills several long prompts at once (largest)
        _append("append_prompts", "bfloat16", 5, (1100, 4001), (0, 37), 32, 32, 128, 64, False),
        # a small fp32 model that continues ragged chunks
        _append("append_fp32", "float32", 9, (1, 333), (0, 700), 12, 12, 64, 24, True),
        # one user's single token against a medium context
        _attend("decode_one", "bfloat16", 1, (1, 1), (2010, 2010), 32, 32, 128, 16),
        # a serving batch of single tokens, ragged contexts up to 8K, grouped heads (largest in bytes)
        _attend("decode_batch", "float16", 64, (1, 1), (300, 8100), 32, 8, 128, 16),
        # one chunk of a long prompt over what is already cached
        _attend("chunk_one", "bfloat16", 1, (501, 501), (7600, 7600), 32, 8, 128, 64),
        # prompts from an empty cache (largest in operations)
        _attend("prefill", "bfloat16", 2, (3700, 4096), (0, 0), 32, 32, 128, 64),
        # a mixed step of a small model: decoding sequences beside short chunks
        _attend("mixed", "float16", 24, (1, 96), (5, 1500), 12, 12, 64, 16),
        # one user's next token
        _sample("sample_one", "bfloat16", 1, 32000, 0.8, 50, 0.95, 0.0),
        # a batch whose requests each bring their own settings
        _sample("sample_mixed", "bfloat16", 256, 32000, 1.0, 0, 1.0, 0.0, True),
        # nucleus sampling over a large fp32 vocabulary (largest)
        _sample("sample_wide", "float32", 192, 131072, 1.0, 0, 0.9, 0.0),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _some(rng, lo, hi):
    """A range within [lo, hi], as (low, high)."""
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return (min(a, b), max(a, b))


def draw(rng: random.Random):
    op = rng.choice(["append", "attention", "attention", "sample"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "sample":
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        vocab = _log(rng, 1000, 131072)
        rows = _log(rng, 1, min(256, 24_000_000 // vocab))
        if rng.random() < 0.4:
            c = _sample("", dtype, rows, vocab, 1.0, 0, 1.0, 0.0, True)
        else:
            c = _sample("", dtype, rows, vocab, round(rng.uniform(0.3, 1.5), 3),
                        rng.choice([0, 0, 1, _log(rng, 2, 400)]),
                        rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                        rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]))
    else:
        heads, kv = rng.choice([(32, 32), (32, 8), (12, 12), (8, 1), (6, 2)])
        dim = rng.choice([64, 128])
        page = rng.choice([8, 16, 24, 32, 64, 128])
        kind = rng.choice(["decode", "mixed", "chunk"])
        if kind == "decode":
            seqs = _log(rng, 1, 128)
            new, old = (1, 1), _some(rng, 1, 8000 if op == "append" else max(2, min(8000, 400_000 // seqs)))
        elif kind == "mixed":
            seqs = _log(rng, 2, 32)
            new, old = _some(rng, 1, 64), _some(rng, 1, min(4000, 60_000 // seqs))
        else:
            seqs = _log(rng, 1, 4)
            new, old = _some(rng, 65, 2000 // seqs), _some(rng, 1, 4000)
        if op == "append":
            dtype = rng.choice(["bfloat16", "float16", "float32"])
            c = _append("", dtype, seqs, new, old, heads, kv, dim, page, rng.random() < 0.5)
        else:
            c = _attend("", dtype, seqs, new, old, heads, kv, dim, page, rng.random() < 0.8)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, keys already there) of each sequence, spread evenly over the case's ranges."""
    b, last = case["seqs"], max(case["seqs"] - 1, 1)
    new = [case["new_hi"] - (case["new_hi"] - case["new_lo"]) * i // last for i in range(b)]
    old = [case["old_hi"] - (case["old_hi"] - case["old_lo"]) * ((5 * i + 2) % b) // last
           for i in range(b)]
    return new, old


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (4 + 8 + (16 if case["mixed"] else 0)),
                "flops": 4 * n}
    new, old = _lengths(case)
    n, h, hkv, d = sum(new), case["heads"], case["kv_heads"], case["head_dim"]
    lists = 4 * (2 * len(new) + 1)
    if case["op"] == "append":
        # page numbers and table rows of each token are read once
        return {"bytes": 2 * n * (h + 2 * hkv) * d * e + n * (4 + 4 * d) + lists,
                "flops": 3 * n * (h + hkv) * d}
    keys = sum(a + b for a, b in zip(new, old))
    pages = sum(-(-(a + b) // case["page"]) for a, b in zip(new, old))
    seen = sum(a * b + a * (a + 1) // 2 if case["causal"] else a * (a + b) for a, b in zip(new, old))
    return {"bytes": 2 * n * h * d * e + 2 * keys * hkv * d * e + 4 * pages + lists,
            "flops": 4 * h * d * seen}


# ------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few clear favourites over a broad tail, some rows sharper than others
        logits = torch.randn(rows, vocab, device="cuda", generator=g) * (0.8 + 2.2 * uniform(rows, 1))
        logits = logits.to(dt)
        s = {"op": "sample", "logits": logits, "u": uniform(rows)}
        if case["mixed"]:
            kind = torch.randint(0, 4, (4, rows), device="cuda", generator=g)
            s["temperature"] = torch.where(kind[0] == 0, 0.0, 0.4 + uniform(rows))
            s["top_k"] = torch.where(kind[1] < 2, 0, 1 + (uniform(rows) * 100).int()).int()
            s["top_p"] = torch.where(kind[2] < 1, 1.0, 0.6 + 0.39 * uniform(rows))
            s["min_p"] = torch.where(kind[3] < 3, 0.0, 0.01 + 0.1 * uniform(rows))
        else:
            for name in ("temperature", "top_k", "top_p", "min_p"):
                s[name] = case[name]
        return s

    new, old = _lengths(case)
    order = torch.randperm(len(new), device="cuda", generator=g).tolist()
    new, old = [new[i] for i in order], [old[i] for i in order]
    lens = [a + b for a, b in zip(new, old)]
    h, hkv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    n, most = sum(new), max(-(-x // page) for x in lens)
    used = [-(-x // page) for x in lens]
    pages = sum(used) + 3
    shuffled = torch.randperm(pages, device="cuda", generator=g).int()
    starts = torch.tensor([sum(used[:i]) for i in range(len(used))], device="cuda")
    at = starts[:, None] + torch.arange(most, device="cuda")
    table = shuffled[at.clamp(max=pages - 1)].contiguous()
    s = {"op": case["op"], "page_table": table,
         "cu_q": torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda"),
         "kv_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "k_cache": normal(pages, hkv, page, d), "v_cache": normal(pages, hkv, page, d)}
    if case["op"] == "attention":
        s.update(q=normal(n, h, d), causal=case["causal"], max_new=max(new), max_len=max(lens))
        return s
    if case["fused"]:  # the three are views of one projection's rows
        qkv = normal(n, h + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    else:
        s["q"], s["k"], s["v"] = normal(n, h, d), normal(n, hkv, d), normal(n, hkv, d)
    inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.outer(torch.arange(_MAX_POSITIONS, device="cuda", dtype=torch.float64), inv)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        from autokernel_b200 import ops
        if s["op"] == "append":
            q = ops.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"],
                                 s["cu_q"], s["kv_lens"], q=s["q"], cos=s["cos"], sin=s["sin"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"],
                                       s["cu_q"], s["kv_lens"], causal=s["causal"])
        return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"])
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[s["op"]](s)


def _positions(s, n):
    """Sequence and position of each of the n packed tokens."""
    cu = s["cu_q"].long()
    i = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    return seq, s["kv_lens"].long()[seq] - (cu[seq + 1] - i)


def _rotate(x, cos, sin):
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)


def _plain_append(s):
    seq, pos = _positions(s, s["k"].shape[0])
    size = s["k_cache"].shape[2]
    page = s["page_table"].long()[seq, pos // size]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["k_cache"][page, :, pos % size] = _rotate(s["k"], cos, sin)
    s["v_cache"][page, :, pos % size] = s["v"]
    return {"q": _rotate(s["q"], cos, sin), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    q, cu, lens = s["q"], s["cu_q"].long(), s["kv_lens"].long()
    n, h, d = q.shape
    b, (_, hkv, size, _) = lens.numel(), s["k_cache"].shape
    group, new, length = h // hkv, s["max_new"], s["max_len"]
    pages = s["page_table"][:, :-(-length // size)].long()

    def padded(cache):  # [B, Hkv, length, D]
        return cache[pages].transpose(1, 2).reshape(b, hkv, -1, d)[:, :, :length].float()

    t = torch.arange(new, device=q.device)
    x = q[(cu[:-1, None] + t).clamp(max=n - 1)].float().view(b, new, hkv, group, d)
    x = x.permute(0, 2, 3, 1, 4).reshape(b, hkv, group * new, d)
    score = (x @ padded(s["k_cache"]).transpose(-1, -2)) * d ** -0.5
    seen = (lens - (cu[1:] - cu[:-1]))[:, None] + t + 1 if s["causal"] else lens[:, None].expand(b, new)
    hidden = torch.arange(length, device=q.device) >= seen[..., None]  # [B, new, length]
    score = score.view(b, hkv * group, new, length).masked_fill_(hidden[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = score.sum(-1, keepdim=True).view(b, hkv, group * new, 1)
    out = score.view(b, hkv, group * new, length) @ padded(s["v_cache"])
    out = torch.where(total > 0, out / total, 0.0).view(b, h, new, d)
    i = torch.arange(n, device=q.device)
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    return out[seq, :, i - cu[seq]].to(q.dtype)


def _per_row(v, rows, device):
    """A setting of each row in 64 bits, from the 32 bits in which it is given."""
    if not isinstance(v, torch.Tensor):
        v = torch.full((rows,), v, dtype=torch.float32, device=device)
    return v.double()[:, None]


def _plain_sample(s):
    x, u = s["logits"].double(), s["u"].double()[:, None]
    rows, vocab = x.shape
    t, k, p, m = (_per_row(s[name], rows, x.device) for name in ("temperature", "top_k", "top_p", "min_p"))
    x, index = x.sort(dim=-1, descending=True, stable=True)
    weight = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(vocab, device=x.device)
    weight = torch.where((k <= 0) | (rank < k), weight, 0.0)
    before = torch.cat((torch.zeros_like(u), weight.cumsum(-1)), -1)
    kept = (before[:, :-1] < p * before[:, -1:]) | (p >= 1) | (rank == 0)
    weight = torch.where(kept & (weight >= m), weight, 0.0)
    weight = torch.zeros_like(weight).scatter(1, index, weight)  # back in the vocabulary's order
    total = weight.cumsum(-1)
    past = total > u * total[:, -1:]
    chosen = past.long().argmax(-1)
    return torch.where(t[:, 0] > 0, chosen, index[:, 0])


# ------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "sample":
        return _exact_sample(s)
    lens, cu = s["kv_lens"].tolist(), s["cu_q"].tolist()
    size = s["k_cache"].shape[2]
    table = s["page_table"].long()
    if s["op"] == "append":
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        turn = torch.complex(s["cos"].double(), s["sin"].double())

        def turned(x, at):
            z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous())
            return torch.view_as_real(z * turn[at][:, None]).reshape(x.shape)

        out = []
        for b, length in enumerate(lens):
            rows = slice(cu[b], cu[b + 1])
            at = torch.arange(length - (cu[b + 1] - cu[b]), length, device="cuda")
            page, slot = table[b][at.div(size, rounding_mode="floor")], at.remainder(size)
            k_cache[page, :, slot] = turned(s["k"][rows], at)
            v_cache[page, :, slot] = s["v"][rows].double()
            out.append(turned(s["q"][rows], at))
        return {"q": torch.cat(out), "k_cache": k_cache, "v_cache": v_cache}
    _, h, d = s["q"].shape
    hkv = s["k_cache"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        new = cu[b + 1] - cu[b]
        at = torch.arange(length, device="cuda")
        page, slot = table[b][at.div(size, rounding_mode="floor")], at.remainder(size)
        last = torch.arange(length - new, length, device="cuda")[:, None]
        for head in range(h):
            k = s["k_cache"][page, head * hkv // h, slot].double()
            v = s["v_cache"][page, head * hkv // h, slot].double()
            z = torch.einsum("td,sd->ts", s["q"][cu[b]:cu[b + 1], head].double(), k) / d ** 0.5
            if s["causal"]:
                z = z.masked_fill(at > last, float("-inf"))
            out[cu[b]:cu[b + 1], head] = torch.softmax(z, -1) @ v
    return out


def _exact_sample(s):
    rows, vocab = s["logits"].shape
    settings = []
    for name in ("temperature", "top_k", "top_p", "min_p"):
        v = s[name]
        v = v if isinstance(v, torch.Tensor) else torch.tensor([v] * rows, dtype=torch.float32)
        settings.append(v.double().tolist())
    tokens = []
    for r, (t, k, p, m) in enumerate(zip(*settings)):
        x = s["logits"][r].double()
        if t == 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            continue
        order = torch.argsort(-x, stable=True)
        keep = order[: int(k)] if k > 0 else order
        prob = torch.softmax(x[keep] / t, 0)
        if p < 1:
            ahead = prob.cumsum(0) - prob
            keep, prob = keep[ahead < p], prob[ahead < p]
        keep = keep[prob >= m * prob[0]]
        keep = keep.sort().values
        share = torch.softmax(x[keep] / t, 0).cumsum(0)
        at = int(torch.searchsorted(share, share[-1:] * s["u"][r].double(), right=True)[0])
        tokens.append(int(keep[min(at, keep.numel() - 1)]))
    return torch.tensor(tokens)
