"""LlamaB200.generate's bookkeeping on the CPU: a model whose next token is the last one + 1, and a sampler that
takes the likeliest, in place of the kernels."""
from __future__ import annotations

import pytest
import torch

from autokernel_b200 import AkError, ops
from autokernel_b200.llama import LlamaB200, LlamaConfig

VOCAB = 100


class Counting(LlamaB200):
    """extend() returns logits whose largest is that of the last token + 1, and checks the batch."""

    def __init__(self):
        cfg = LlamaConfig(vocab_size=VOCAB, dim=8, n_layers=1, n_heads=1, n_kv_heads=1, hidden_dim=8)
        super().__init__(cfg, {"tok_embeddings.weight": torch.zeros(VOCAB, 8)})

    def extend(self, tokens, batch, cache):
        assert tokens.shape == (batch.n_tokens,)
        last = tokens[batch.cu_q[1:].long() - 1]
        return torch.nn.functional.one_hot((last + 1) % VOCAB, VOCAB).float()


@pytest.fixture
def settings(monkeypatch):
    """The settings of every ops.sample call, each as one number per row."""
    seen = []

    def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        n = logits.shape[0]
        row = [v.tolist() if isinstance(v, torch.Tensor) else [v] * n for v in (temperature, top_k, top_p, min_p)]
        assert all(len(r) == n for r in row)
        seen.append([tuple(x) for x in zip(*row)])
        return logits.argmax(-1)

    monkeypatch.setattr(ops, "sample", sample)
    return seen


def test_a_stopped_sequence_gives_its_pages_back_at_once(settings):
    """8 pages of 4: the first two answers stop after one token, and the third grows into their pages."""
    m = Counting()
    cache = m.new_cache(8, 4)
    got = m.generate([[41] * 12, [41] * 8, [1, 2, 3]], 20, stop=42, cache=cache)
    assert got == [[42], [42], list(range(4, 24))]
    assert cache.free_pages == 8


def test_a_full_cache_does_not_lose_the_answers_so_far(settings):
    """3 pages of 4: the second sequence's fifth key finds no page; what was sampled by then comes with the error."""
    m = Counting()
    cache = m.new_cache(3, 4)
    with pytest.raises(AkError, match="full") as e:
        m.generate([[10, 11, 12, 13, 14], [30, 31]], 20, cache=cache)
    assert e.value.answers == [[15, 16, 17], [32, 33, 34]]
    assert cache.free_pages == 3
    with pytest.raises(AkError, match="full") as e:
        m.generate([[1] * 13], 20, cache=cache)
    assert e.value.answers == [[]]
    assert cache.free_pages == 3


@pytest.mark.parametrize("kind", ["list", "tensor"])
def test_settings_of_each_prompt_follow_their_sequences(settings, kind):
    """The second and then the first sequence stop: each row keeps the settings of its prompt."""
    m = Counting()
    given = dict(temperature=[0.5, 0.25, 2.0], top_k=[1, 0, 7], top_p=[1.0, 0.5, 0.75], min_p=[0.0, 0.125, 0.25])
    if kind == "tensor":
        given = {k: torch.tensor(v) for k, v in given.items()}
    got = m.generate([[38], [40], [1]], 5, stop=41, **given)
    assert got == [[39, 40, 41], [41], [2, 3, 4, 5, 6]]
    rows = list(zip([0.5, 0.25, 2.0], [1, 0, 7], [1.0, 0.5, 0.75], [0.0, 0.125, 0.25]))
    assert settings == [rows, [rows[0], rows[2]], [rows[0], rows[2]], [rows[2]], [rows[2]]]


def test_bad_settings_are_refused_before_anything_is_run(settings):
    m = Counting()
    cache = m.new_cache(4, 4)
    for bad in (dict(temperature=[1.0]), dict(top_p=torch.ones(3)), dict(min_p=torch.ones(2, 1)), dict(top_k=[1, -1]),
                dict(temperature=[0.5, float("nan")]), dict(top_k=torch.ones(2)), dict(top_p=-0.5)):
        with pytest.raises(ValueError):
            m.generate([[1], [2]], 3, cache=cache, **bad)
    assert settings == [] and cache.free_pages == 4


def test_tokens_outside_of_the_vocabulary_embed_as_nan():
    """A gather with such an index ends the CUDA context; extend() has to take whatever a sampler gave (-1 too)."""
    m = Counting()
    m.w["tok_embeddings.weight"] = torch.arange(VOCAB * 8).view(VOCAB, 8).half()
    for dt in (torch.int64, torch.int32):
        h = m._embed(torch.tensor([3, -1, 99, 100, 2 ** 31 - 1, -2 ** 31, 0], dtype=dt))
        assert h.dtype == torch.float16 and h.isnan().all(-1).tolist() == [False, True, False, True, True, True, False]
        assert torch.equal(h[[0, 2, 6]], m.w["tok_embeddings.weight"][[3, 99, 0]])
