"""LLaMA forward (+ next-token cross entropy) on the nine B200 operators.

The architecture is AutoKernel's models/llama_7b.py (LlamaModel / LlamaModel7B,
models/llama_7b.py:114-209): token embedding, n_layers x [RMSNorm -> q/k/v
projections -> interleaved RoPE -> causal attention (grouped KV heads) -> output
projection -> residual; RMSNorm -> SwiGLU MLP -> residual], final RMSNorm, LM head.
Parameter names are the reference module's state_dict keys, so
`LlamaB200.from_state_dict(ref_model.state_dict(), cfg)` runs a reference model's
weights unchanged.  This is the model-level drop-in that verify.py performs by
module surgery (verify.py:510-641), extended to attention, RoPE, the MLP and the
loss.

Every arithmetic step is one of this package's kernels:
    RMSNorm              folded into the projections that read it (16-bit weights): the
                         o-/down-projection epilogues write per-row sums of squares of the
                         new hidden state, the q/k/v and gate/up GEMMs scale their rows by
                         1 / rms with the norm weight folded into their weights, so the
                         normalised activations are never stored (ops.linear_rms,
                         ops.mlp_hidden_rms); otherwise ops.rmsnorm_fp32 (csrc/rowops.cu)
    q/k/v/o projections  ops.linear            (tcgen05 GEMM, K-major weights, no copies)
    RoPE                 ops.rope_apply        (fp32 cos/sin table, [B, T, H, D] in place)
    attention            ops.attention_bhsd    (reads [B, T, H, D] views, GQA, causal)
    SwiGLU MLP           ops.mlp_hidden + ops.linear (dual GEMM + SiLU*mul epilogue, down GEMM)
    residual adds        in the o-projection / down-projection GEMM epilogues, in place
    LM head + loss       ops.linear_cross_entropy_partial: one tcgen05 GEMM whose epilogue
                         reduces each vocab tile to (max, sum exp) and the target logit
                         (the logits are never stored; ignore_index masks the last position)
Glue left to torch: the embedding gather.

Answering (extend, generate) runs the same layers over a paged cache of keys and values
(paged.PagedCache): the projections' q and k are rotated and k, v stored by ops.paged_append,
the new tokens attend by ops.paged_attention, and ops.sample draws the next token.
"""
from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch

from . import ops, shard
from ._lib import AkError
from .paged import Batch, CacheFull, PagedCache


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    dim: int = 4096
    n_layers: int = 32
    n_heads: int = 32
    n_kv_heads: int = 32
    hidden_dim: int = 11008
    norm_eps: float = 1e-6
    rope_theta: float = 10000.0

    @property
    def head_dim(self) -> int:
        return self.dim // self.n_heads

    def linear_params(self) -> int:
        hd = self.head_dim
        per_layer = (self.dim * self.n_heads * hd + 2 * self.dim * self.n_kv_heads * hd
                     + self.n_heads * hd * self.dim + 3 * self.dim * self.hidden_dim)
        return self.n_layers * per_layer + self.dim * self.vocab_size

    def flops_per_token(self, seq_len: int) -> float:
        """Forward FLOPs per token: 2 x linear params + causal attention (QK^T and PV over the
        (T+1)/2 visible keys on average)."""
        attn = self.n_layers * 2 * 2 * self.n_heads * self.head_dim * (seq_len + 1) / 2
        return 2.0 * self.linear_params() + attn


LLAMA_7B = LlamaConfig()  # BASELINE e2e config: 32 heads of 128, MHA (n_kv_heads = 32)


def rope_tables(seq_len: int, head_dim: int, theta: float, device):
    """fp32 cos/sin [T, 1, head_dim/2] of angle t * theta^(-2i/head_dim), the table
    precompute_freqs_cis builds (models/llama_7b.py:33-37), shaped to broadcast over heads."""
    inv = 1.0 / theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim)
    ang = torch.outer(torch.arange(seq_len, device=device, dtype=torch.float32), inv)
    return ang.cos()[:, None, :].contiguous(), ang.sin()[:, None, :].contiguous()


class LlamaB200:
    """Inference-mode LLaMA whose forward runs on the autokernel_b200 kernels."""

    def __init__(self, cfg: LlamaConfig, weights: dict[str, torch.Tensor],
                 fuse_norms: bool | None = None):
        self.cfg = cfg
        self.w = weights
        self._rope: dict = {}
        dt = weights["tok_embeddings.weight"].dtype
        # RMSNorm folded into the projections after it (16-bit weights: tensor-core GEMMs)
        self.fuse_norms = dt in (torch.float16, torch.bfloat16) if fuse_norms is None else fuse_norms
        # with folded norms, RoPE of q and k runs in their projection GEMMs' epilogue
        self.fuse_rope = self.fuse_norms
        self._folded: dict[int, tuple] = {}

    @staticmethod
    def random_weights(cfg: LlamaConfig, device, dtype=torch.float16, seed: int = 0,
                       std: float = 0.02) -> dict[str, torch.Tensor]:
        """N(0, std) linear / embedding weights and unit norms (BASELINE: fp16, N(0, 0.02))."""
        g = torch.Generator(device=device).manual_seed(seed)
        hd = cfg.head_dim

        def rnd(*shape):
            return (torch.randn(*shape, device=device, generator=g) * std).to(dtype)

        w = {"tok_embeddings.weight": rnd(cfg.vocab_size, cfg.dim)}
        for i in range(cfg.n_layers):
            p = f"layers.{i}."
            w[p + "attention.wq.weight"] = rnd(cfg.n_heads * hd, cfg.dim)
            w[p + "attention.wk.weight"] = rnd(cfg.n_kv_heads * hd, cfg.dim)
            w[p + "attention.wv.weight"] = rnd(cfg.n_kv_heads * hd, cfg.dim)
            w[p + "attention.wo.weight"] = rnd(cfg.dim, cfg.n_heads * hd)
            w[p + "feed_forward.w1.weight"] = rnd(cfg.hidden_dim, cfg.dim)
            w[p + "feed_forward.w2.weight"] = rnd(cfg.dim, cfg.hidden_dim)
            w[p + "feed_forward.w3.weight"] = rnd(cfg.hidden_dim, cfg.dim)
            w[p + "attention_norm.weight"] = torch.ones(cfg.dim, device=device, dtype=dtype)
            w[p + "ffn_norm.weight"] = torch.ones(cfg.dim, device=device, dtype=dtype)
        w["norm.weight"] = torch.ones(cfg.dim, device=device, dtype=dtype)
        w["output.weight"] = rnd(cfg.vocab_size, cfg.dim)
        return w

    @classmethod
    def from_state_dict(cls, sd: dict, cfg: LlamaConfig, device="cuda", dtype=torch.float16):
        """Weights of a reference LlamaModel / LlamaModel7B (its state_dict keys)."""
        w = {k: v.detach().to(device=device, dtype=dtype).contiguous()
             for k, v in sd.items() if not k.endswith("freqs_cis")}
        return cls(cfg, w)

    def _tables(self, T: int, device):
        key = (T, str(device))
        if key not in self._rope:
            self._rope[key] = rope_tables(T, self.cfg.head_dim, self.cfg.rope_theta, device)
        return self._rope[key]

    def _layer(self, i: int, h: torch.Tensor, cos, sin) -> torch.Tensor:
        c, w = self.cfg, self.w
        p = f"layers.{i}."
        B, T, _ = h.shape
        hd = c.head_dim
        x = ops.rmsnorm_fp32(h, w[p + "attention_norm.weight"], c.norm_eps)
        q = ops.linear(x, w[p + "attention.wq.weight"]).view(B, T, c.n_heads, hd)
        k = ops.linear(x, w[p + "attention.wk.weight"]).view(B, T, c.n_kv_heads, hd)
        v = ops.linear(x, w[p + "attention.wv.weight"]).view(B, T, c.n_kv_heads, hd)
        q = ops.rope_apply(q, cos, sin)
        k = ops.rope_apply(k, cos, sin)
        o = self._attention(q, k, v, B, T)
        # residual adds happen in the GEMM epilogues, in place on h
        ops.linear(o.view(B, T, c.n_heads * hd), w[p + "attention.wo.weight"], residual=h, out=h)
        x = ops.rmsnorm_fp32(h, w[p + "ffn_norm.weight"], c.norm_eps)
        hidden = ops.mlp_hidden(x, w[p + "feed_forward.w1.weight"], w[p + "feed_forward.w3.weight"])
        ops.linear(hidden, w[p + "feed_forward.w2.weight"], residual=h, out=h)
        return h

    def _fold(self, i: int) -> tuple:
        """Projection weights of layer i with the RMSNorm weight that precedes them folded in
        (w * diag(norm.weight), rounded once): q, k, v after attention_norm, w1, w3 after
        ffn_norm.  Built once; the reference weights are kept for the unfused path."""
        if i not in self._folded:
            w, p = self.w, f"layers.{i}."
            an, fn = w[p + "attention_norm.weight"], w[p + "ffn_norm.weight"]
            self._folded[i] = tuple(
                ops.fold_norm_weight(w[p + k], n) for k, n in (
                    ("attention.wq.weight", an), ("attention.wk.weight", an),
                    ("attention.wv.weight", an), ("feed_forward.w1.weight", fn),
                    ("feed_forward.w3.weight", fn)))
        return self._folded[i]

    def _attention(self, q, k, v, B, T):
        c = self.cfg
        hd = c.head_dim
        o = torch.empty(B, T, c.n_heads, hd, dtype=q.dtype, device=q.device)
        r = ops.attention_bhsd(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                               causal=True, out=o.transpose(1, 2))
        if r is None:  # layouts / head sizes the tensor-core path cannot take
            rep = c.n_heads // c.n_kv_heads
            o = ops.flash_attention(q.transpose(1, 2),
                                    k.transpose(1, 2).repeat_interleave(rep, 1),
                                    v.transpose(1, 2).repeat_interleave(rep, 1))
            o = o.transpose(1, 2).contiguous()
        return o

    def _layer_fused(self, i: int, h: torch.Tensor, ss: torch.Tensor, cos, sin):
        """One decoder layer with both RMSNorms folded into the GEMMs that read them: ss holds
        the per-row partial sums of squares of h, and the o-projection and down-projection
        epilogues (which add the residual into h in place) write those of the new h."""
        c, w = self.cfg, self.w
        p = f"layers.{i}."
        B, T, _ = h.shape
        hd, eps = c.head_dim, c.norm_eps
        wq, wk, wv, w1, w3 = self._fold(i)
        rope = (cos, sin, T, hd) if self.fuse_rope else None
        q = ops.linear_rms(h, wq, ss, eps, rope=rope).view(B, T, c.n_heads, hd)
        k = ops.linear_rms(h, wk, ss, eps, rope=rope).view(B, T, c.n_kv_heads, hd)
        v = ops.linear_rms(h, wv, ss, eps).view(B, T, c.n_kv_heads, hd)
        if not self.fuse_rope:
            q = ops.rope_apply(q, cos, sin)
            k = ops.rope_apply(k, cos, sin)
        o = self._attention(q, k, v, B, T)
        _, ss = ops.linear_rms(o.view(B, T, c.n_heads * hd), w[p + "attention.wo.weight"],
                               residual=h, out=h, want_ss=True)
        hidden = ops.mlp_hidden_rms(h, w1, w3, ss, eps)
        _, ss = ops.linear_rms(hidden, w[p + "feed_forward.w2.weight"], residual=h, out=h,
                               want_ss=True)
        return h, ss

    @torch.no_grad()
    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        """The final normalised hidden state [B, T, dim], the LM head's input."""
        _, T = tokens.shape
        cos, sin = self._tables(T, tokens.device)
        h = torch.nn.functional.embedding(tokens, self.w["tok_embeddings.weight"])  # new tensor
        if self.fuse_norms:
            ss = ops.row_sumsq(h)
            for i in range(self.cfg.n_layers):
                h, ss = self._layer_fused(i, h, ss, cos, sin)
        else:
            for i in range(self.cfg.n_layers):
                h = self._layer(i, h, cos, sin)
        return ops.rmsnorm_fp32(h, self.w["norm.weight"], self.cfg.norm_eps)

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits [B, T, vocab] (models/llama_7b.py:199-209)."""
        return ops.linear(self.hidden(tokens), self.w["output.weight"])

    __call__ = forward

    # ------------------------------------------------------------ over a paged cache

    def new_cache(self, num_pages: int, page_size: int = 64) -> PagedCache:
        """A paged cache for this model's layers, in its dtype and on its device."""
        e = self.w["tok_embeddings.weight"]
        return PagedCache(self.cfg.n_layers, self.cfg.n_kv_heads, self.cfg.head_dim, num_pages, page_size,
                          e.dtype, e.device)

    def _cached_attention(self, i: int, q, k, v, batch: Batch, cache: PagedCache, cos, sin) -> torch.Tensor:
        """q [N, n_heads * hd] and k, v [N, n_kv_heads * hd] of layer i's new tokens: rotate q and k, store
        k and v, attend."""
        c, N = self.cfg, q.shape[0]
        q = q.view(N, c.n_heads, c.head_dim)
        ops.paged_append(k.view(N, c.n_kv_heads, c.head_dim), v.view(N, c.n_kv_heads, c.head_dim),
                         cache.k[i], cache.v[i], *batch.lists, q=q, cos=cos, sin=sin, q_out=q)
        return ops.paged_attention(q, cache.k[i], cache.v[i], *batch.lists).view(N, -1)

    def _embed(self, tokens: torch.Tensor) -> torch.Tensor:
        """The embeddings of tokens [N]; NaN for one that is not in the vocabulary (no host code knows them, and a
        gather outside of the table would end the CUDA context)."""
        table = self.w["tok_embeddings.weight"]
        known = tokens.clamp(0, table.shape[0] - 1)
        return torch.nn.functional.embedding(known, table).masked_fill_((known != tokens)[:, None], float("nan"))

    @torch.no_grad()
    def extend(self, tokens: torch.Tensor, batch: Batch, cache: PagedCache) -> torch.Tensor:
        """Run the packed new tokens [N] of a batch (cache.extend) and return the logits [B, vocab] that
        follow the last one of each sequence.  A token outside of the vocabulary (ops.sample's -1) makes its
        sequence's logits NaN from there on, and no other's."""
        c, w = self.cfg, self.w
        if tokens.shape != (batch.n_tokens,):
            raise ValueError(f"extend: the batch holds {batch.n_tokens} tokens, got {tuple(tokens.shape)}")
        # tables to the next power of two, so that decoding does not rebuild them at every step
        cos, sin = self._tables(max(2048, 1 << (batch.max_len - 1).bit_length()), tokens.device)
        h = self._embed(tokens)
        ss = ops.row_sumsq(h) if self.fuse_norms else None
        for i in range(c.n_layers):
            p = f"layers.{i}."
            wo, w2 = w[p + "attention.wo.weight"], w[p + "feed_forward.w2.weight"]
            if self.fuse_norms:
                wq, wk, wv, w1, w3 = self._fold(i)
                q, k, v = (ops.linear_rms(h, x, ss, c.norm_eps) for x in (wq, wk, wv))
                o = self._cached_attention(i, q, k, v, batch, cache, cos, sin)
                _, ss = ops.linear_rms(o, wo, residual=h, out=h, want_ss=True)
                hidden = ops.mlp_hidden_rms(h, w1, w3, ss, c.norm_eps)
                _, ss = ops.linear_rms(hidden, w2, residual=h, out=h, want_ss=True)
            else:
                x = ops.rmsnorm_fp32(h, w[p + "attention_norm.weight"], c.norm_eps)
                q, k, v = (ops.linear(x, w[p + f"attention.{n}.weight"]) for n in ("wq", "wk", "wv"))
                o = self._cached_attention(i, q, k, v, batch, cache, cos, sin)
                ops.linear(o, wo, residual=h, out=h)
                x = ops.rmsnorm_fp32(h, w[p + "ffn_norm.weight"], c.norm_eps)
                hidden = ops.mlp_hidden(x, w[p + "feed_forward.w1.weight"], w[p + "feed_forward.w3.weight"])
                ops.linear(hidden, w2, residual=h, out=h)
        last = h.index_select(0, batch.cu_q[1:] - 1)
        return ops.linear(ops.rmsnorm_fp32(last, w["norm.weight"], c.norm_eps), w["output.weight"])

    @torch.no_grad()
    def generate(self, prompts: list[list[int]], max_new_tokens: int,
                 temperature: float | Sequence[float] | torch.Tensor = 1.0,
                 top_k: int | Sequence[int] | torch.Tensor = 0, top_p: float | Sequence[float] | torch.Tensor = 1.0,
                 min_p: float | Sequence[float] | torch.Tensor = 0.0, stop: int | None = None,
                 generator: torch.Generator | None = None,
                 cache: PagedCache | None = None) -> list[list[int]]:
        """Continue each prompt (token lists, at least one token each) by up to max_new_tokens sampled
        tokens (ops.sample's settings, each a number or one per prompt; temperature 0 takes the
        likeliest).  A sequence ends with the token `stop`, if given.  All sequences decode together; with
        `cache` they share its pages, each giving its own back when it ends, otherwise one of the right
        size is made.  Raises CacheFull when a step finds no pages, with the tokens sampled so far as its
        `answers`, and AkError when a step's logits held nothing to draw (all NaN)."""
        if not prompts or min(len(p) for p in prompts) < 1 or max_new_tokens < 0:
            raise ValueError("generate: need prompts of at least one token")
        vocab = self.w["tok_embeddings.weight"].shape[0]
        if not all(0 <= t < vocab for p in prompts for t in p):
            raise ValueError(f"generate: tokens must lie in [0, {vocab})")
        device = self.w["tok_embeddings.weight"].device
        settings = [_setting(n, v, len(prompts), device) for n, v in (
            ("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p))]
        if max_new_tokens == 0:
            return [[] for _ in prompts]
        if cache is None:
            size = 64
            cache = self.new_cache(sum(-(-(len(p) + max_new_tokens) // size) for p in prompts), size)
        live = list(range(len(prompts)))
        seqs = {i: cache.add() for i in live}  # those that hold pages
        tokens = torch.tensor([t for p in prompts for t in p], device=device)
        counts = [len(p) for p in prompts]
        steps: list[tuple[list[int], torch.Tensor]] = []

        def answers() -> list[list[int]]:
            out: list[list[int]] = [[] for _ in prompts]
            for rows, t in steps:
                for i, x in zip(rows, t.tolist()):
                    if x < 0:
                        raise AkError(f"generate: sequence {i} has no logits to draw from")
                    out[i].append(x)
            return out

        try:
            for _ in range(max_new_tokens):
                batch = cache.extend([seqs[i] for i in live], counts)
                logits = self.extend(tokens, batch, cache)
                u = torch.rand(len(live), device=device, generator=generator)
                tokens = ops.sample(logits, u, *settings)
                steps.append((live, tokens))
                tokens = tokens.clamp(min=0)  # -1: nothing to draw, found when the answers are read
                if stop is not None:
                    on = (tokens != stop).tolist()
                    if not all(on):
                        rest = torch.tensor(on, device=device)
                        tokens = tokens[rest]
                        settings = [v[rest] if isinstance(v, torch.Tensor) else v for v in settings]
                    for i, x in zip(live, on):
                        if not x:
                            cache.release(seqs.pop(i))
                    live = [i for i, x in zip(live, on) if x]
                    if not live:
                        break
                counts = [1] * len(live)
        except CacheFull as e:
            e.answers = answers()
            raise
        finally:
            for s in seqs.values():
                cache.release(s)
        return answers()

    @staticmethod
    def next_token_targets(tokens: torch.Tensor) -> torch.Tensor:
        """Targets [B, T]: tokens shifted left by one, the last position ignored (-100), so the
        loss over all B*T logit rows equals the mean over the B*(T-1) predicted positions."""
        t = torch.full_like(tokens, ops.IGNORE_INDEX)
        t[:, :-1] = tokens[:, 1:]
        return t

    @torch.no_grad()
    def loss(self, tokens: torch.Tensor, group=None) -> torch.Tensor:
        """Mean next-token cross entropy; with a process group, the mean over all ranks'
        sequences (one fp64 all-reduce of (sum, count)).  The LM head and the loss run as one
        fused kernel (ops.linear_cross_entropy_rows): the [B*T, vocab] logits are never
        stored."""
        h = self.hidden(tokens)
        targets = self.next_token_targets(tokens)
        W = self.w["output.weight"]
        return shard.cross_entropy_sharded(
            h.view(-1, h.shape[-1]), targets.view(-1), group=group,
            partial_fn=lambda x, t: ops.linear_cross_entropy_partial(x, W, t),
            out_dtype=h.dtype)


def _setting(name: str, v, n: int, device) -> float | torch.Tensor:
    """A sampling setting of n prompts as ops.sample takes it: the number, or a tensor [n] of one each."""
    dtype = torch.int32 if name == "top_k" else torch.float32
    if isinstance(v, torch.Tensor):
        if v.shape != (n,) or v.is_floating_point() != dtype.is_floating_point:
            raise ValueError(f"generate: a tensor of {name} must hold one {dtype} per prompt ({n})")
        return v.to(device=device, dtype=dtype)
    numbers = list(v) if isinstance(v, Sequence) else [v]
    if isinstance(v, Sequence) and len(numbers) != n:
        raise ValueError(f"generate: {len(numbers)} values of {name} for {n} prompts")
    if not all(x >= 0 for x in numbers):
        raise ValueError(f"generate: {name} must not be negative, got {v}")
    if isinstance(v, Sequence):
        if name == "top_k":
            numbers = [min(int(x), 2 ** 31 - 1) for x in numbers]
        return torch.tensor(numbers, dtype=dtype, device=device)
    return v


def model_flops(cfg: LlamaConfig, batch: int, seq_len: int) -> float:
    return cfg.flops_per_token(seq_len) * batch * seq_len


__all__ = ["LlamaConfig", "LLAMA_7B", "LlamaB200", "rope_tables", "model_flops"]
