"""What the serving loop refuses on the host, before anything is launched: a position or a token out of
its table's range would be an out-of-range index on the device, which ends the CUDA context."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from vibeblade_b200 import formats as F
from vibeblade_b200 import generate
from vibeblade_b200.engine import LayerConfig
from vibeblade_b200.generate import Decoder

VOCAB, HIDDEN = 50, 128


class Layer:
    """Stands for a DeviceLayer on the CPU: the attention's output is all it passes on."""
    dev, kv_heads = torch.device("cpu"), 1
    cfg = LayerConfig(hidden=HIDDEN, n_heads=2, n_kv_heads=1, ffn=64)

    def forward(self, x, attention):
        q = torch.ones(x.shape[0], HIDDEN)
        return x + attention(q, q[:, :64], q[:, :64])

    def _mm(self, h, w, K, N, t, prefill):
        return h @ w.view(torch.float32)


def decoder(max_tokens=100, vocab=VOCAB, rows=VOCAB, page=16):
    head = torch.zeros(HIDDEN, vocab).view(torch.uint8)
    return Decoder([Layer()], torch.zeros(rows, HIDDEN), torch.ones(HIDDEN), (head, F.GGML_TYPE_F32, vocab), pages=8,
                   page=page, max_tokens=max_tokens)


@pytest.fixture
def no_launch(monkeypatch):
    def fail(*a, **k):
        raise AssertionError("launched")
    for name in ("kv_reserve", "kv_append", "kv_attention", "kv_fork", "token_logprobs"):
        monkeypatch.setattr(generate, name, fail)


def test_lengths_past_max_tokens(no_launch):
    d = decoder()
    for call in (lambda: d.score([[1] * 101]), lambda: d.score([[1], [1] * 101, [2]]),
                 lambda: d.beam_search([1] * 101, 2, 1), lambda: d.beam_search([1] * 90, 2, 12)):
        with pytest.raises(RuntimeError, match="max_tokens"):
            call()
    for call in (lambda: d.score([[1] * 100]), lambda: d.beam_search([1] * 90, 2, 11)):  # the last token is not run
        with pytest.raises(AssertionError, match="launched"):
            call()


@pytest.mark.parametrize("length,new", [(95, 5), (100, 4), (111, 1), (112, 1), (300, 2)])
def test_positions_stay_in_the_table(monkeypatch, length, new):
    """Rows longer than the tables, which only forward's caller can make: the pages are missing, and
    the positions end at the last one there is."""
    d = decoder()
    lens = torch.tensor([length], dtype=torch.int32)
    monkeypatch.setattr(generate, "kv_reserve", lambda refs, tables, lens, n, page: (refs, tables, lens + n, torch.ones(1, dtype=torch.int32)))
    monkeypatch.setattr(generate, "kv_append", lambda *a: None)
    monkeypatch.setattr(generate, "kv_attention", lambda q, *a, **k: q)
    rows = d.rows(1)
    rows.lens = lens
    after, x = d.forward(rows, torch.zeros(new, dtype=torch.long), [new])
    assert x.shape == (new, HIDDEN) and after.lens.item() == length + new


@pytest.mark.parametrize("token", [VOCAB, -1, 1 << 40])
def test_tokens_outside_the_vocabulary(no_launch, token):
    d = decoder()
    for call in (lambda: d.score([[1, 2], [3, token]]), lambda: d.beam_search([token, 1], 2, 3)):
        with pytest.raises(RuntimeError, match="vocabulary"):
            call()


def test_searches_that_cannot_be(no_launch):
    d = decoder()
    for prompt, beams, steps, text in (([], 2, 3, "empty"), ([1], 0, 3, "beams"), ([1], 33, 3, "beams")):
        with pytest.raises(RuntimeError, match=text):
            d.beam_search(prompt, beams, steps)
    with pytest.raises(RuntimeError, match="beams"):
        decoder(vocab=5).beam_search([1], 6, 3)  # the first step has five tokens to choose from


def test_embedding_smaller_than_the_vocabulary():
    with pytest.raises(RuntimeError, match="embedding"):
        decoder(vocab=VOCAB, rows=VOCAB - 1)
    decoder(vocab=VOCAB, rows=VOCAB + 14)  # padded rows are no harm


def test_nothing_to_score(no_launch):
    assert decoder().score([]) == []
    assert [t.numel() for t in decoder().score([[], []])] == [0, 0]
