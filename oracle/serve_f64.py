"""Float64 restatement of the serving operators (paged append, paged attention, sampling), written
token by token from their definitions.  The reference has no counterpart; the rotation is that of
reference.py:63-69."""
from __future__ import annotations

import numpy as np


def token_places(page_table, cu_q, kv_lens, n_tokens, num_pages, page_size):
    """For each packed token (sequence, index in it, position, page, slot); None outside every
    sequence, page -1 where the key has none."""
    out = [None] * n_tokens
    for b in range(len(kv_lens)):
        lo, hi = int(cu_q[b]), int(cu_q[b + 1])
        for t in range(lo, min(hi, n_tokens)):
            p = int(kv_lens[b]) - (hi - lo) + (t - lo)
            page, slot = -1, 0
            if p >= 0 and p // page_size < page_table.shape[1]:
                page, slot = int(page_table[b, p // page_size]), p % page_size
                if not 0 <= page < num_pages:
                    page = -1
            out[t] = (b, t - lo, p, page, slot)
    return out


def rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    y = np.empty_like(x)
    y[..., 0::2] = a * cos - b * sin
    y[..., 1::2] = a * sin + b * cos
    return y


def rotate_size(x, cos, sin):
    """What rotate adds up in each element, |x1 c| + |x2 s| or |x1 s| + |x2 c|: the scale of its fp32 rounding."""
    a, b = np.abs(x[..., 0::2]), np.abs(x[..., 1::2])
    y = np.empty_like(x)
    y[..., 0::2] = a * np.abs(cos) + b * np.abs(sin)
    y[..., 1::2] = a * np.abs(sin) + b * np.abs(cos)
    return y


def paged_append(k, v, k_cache, v_cache, page_table, cu_q, kv_lens, q=None, cos=None, sin=None):
    """(k_cache, v_cache, q) after the append; q keeps its values outside every sequence."""
    k_cache, v_cache = k_cache.copy(), v_cache.copy()
    q = None if q is None else q.copy()
    places = token_places(page_table, cu_q, kv_lens, k.shape[0], k_cache.shape[0], k_cache.shape[2])
    for t, w in enumerate(places):
        if w is None:
            continue
        _, _, p, page, slot = w
        turn = lambda x: x  # noqa: E731
        if cos is not None:
            inside = 0 <= p < cos.shape[0]
            turn = lambda x: rotate(x, cos[p], sin[p]) if inside else np.full_like(x, np.nan)  # noqa: E731,B023
        if page >= 0:
            k_cache[page, :, slot] = turn(k[t])
            v_cache[page, :, slot] = v[t]
        if q is not None:
            q[t] = turn(q[t])
    return k_cache, v_cache, q


def paged_attention(q, k_cache, v_cache, page_table, cu_q, kv_lens, causal, scale):
    """(out, weight, spread, rows): out [N, H, D]; weight = softmax . |V| and spread =
    max_j scale sum |q||k_j| [N, H, 1], which scale the rounding bounds; rows marks the tokens of a
    sequence."""
    N, H, D = q.shape
    P, Hkv, S, _ = k_cache.shape
    out, weight = np.zeros((N, H, D)), np.zeros((N, H, D))
    spread, rows = np.zeros((N, H, 1)), np.zeros(N, bool)
    places = token_places(page_table, cu_q, kv_lens, N, P, S)
    for t, w in enumerate(places):
        if w is None:
            continue
        rows[t] = True
        b, _, p, _, _ = w
        vis = max(p + 1, 0) if causal else int(kv_lens[b])
        if vis == 0:
            continue
        pages = [int(page_table[b, j]) if j < page_table.shape[1] else -1 for j in range(-(-vis // S))]
        if any(not 0 <= x < P for x in pages):
            out[t] = np.nan
            continue
        kk = k_cache[pages].transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :vis]
        vv = v_cache[pages].transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :vis]
        for h in range(H):
            kh, vh = kk[h * Hkv // H], vv[h * Hkv // H]
            s = kh @ q[t, h] * scale
            e = np.exp(s - s.max())
            e /= e.sum()
            out[t, h] = e @ vh
            weight[t, h] = e @ np.abs(vh)
            spread[t, h] = (np.abs(kh) @ np.abs(q[t, h])).max() * scale
    return out, weight, spread, rows


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    """Token of one row of float64 logits."""
    x = np.asarray(x, dtype=np.float64)
    alive = ~(np.isnan(x) | (x == -np.inf))
    if not alive.any():
        return -1
    idx = np.flatnonzero(alive)
    order = idx[np.lexsort((idx, -x[idx]))]
    if not temperature > 0:
        return int(order[0])
    top = x[order[0]]
    with np.errstate(invalid="ignore", under="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    n = len(w)
    if not top_p >= 1:
        ahead = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        n = max(1, int(np.sum(ahead < top_p * w.sum()))) if top_p > 0 else 1
    m = min(min_p, 1.0) if min_p > 0 else 0.0
    keep = np.arange(len(w)) < n
    keep &= w >= m
    order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    c = np.cumsum(w)
    u = min(max(float(u), 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    return int(order[np.argmax(c > u * c[-1])])
