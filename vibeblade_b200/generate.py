"""Decoding with DeviceLayer blocks and the 8-bit paged KV cache: scoring and beam search.

What a serving loop does with the pieces, one after the other (the reference's loop is
VibeBladeFast::generate over forward_layer, cpp/src/fast_model.cpp:578-1090, one sequence
and fp32 keys and values on the host):

    kv_reserve                     pages for the step's tokens
    per block: qkv -> RoPE -> kv_append -> kv_attention -> o, ffn      (DeviceLayer.forward)
    lm_head -> token_logprobs      log probabilities and the likeliest tokens
    kv_fork                        rows regrouped by the beams that live on

Rows are sequences; every tensor of the loop stays on the device and no step waits for it (score and
beam_search wait once, for the count of missing pages).

    dec = Decoder(layers, embedding, final_norm, (lm_head, type, vocab), pages=512)
    logprobs = dec.score([prompt_a, prompt_b])
    tokens, scores = dec.beam_search(prompt, beams=4, steps=32)
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import formats as F
from .engine import DECODE_MAX_TOKENS, DeviceLayer, rms_norm
from .kvcache import kv_append, kv_attention, kv_fork, kv_pool, kv_reserve, token_logprobs


@dataclass
class Rows:
    """Sequences in the cache: their page tables and lengths, and the pages' holders."""
    refs: torch.Tensor    # int32 [pages]
    tables: torch.Tensor  # int32 [rows, max_pages]
    lens: torch.Tensor    # int32 [rows]
    missing: torch.Tensor  # int32 [1]: pages that could not be had so far


class Decoder:
    """``layers``: DeviceLayer blocks of one rank and device; ``embedding`` fp32 [vocab, hidden];
    ``final_norm`` fp32 [hidden]; ``lm_head`` (weight bytes, type, vocab), a hidden x vocab
    matrix.  ``pages`` pages of ``page`` tokens hold the keys and values of every layer, up to
    ``max_tokens`` a row.

    Calls of more than DECODE_MAX_TOKENS rows in all (prompts) run their matmuls on bf16 inputs, and
    their attention on bf16 queries with a bf16 result, so that it takes the tcgen05 kernel; up to as
    many rows everything is fp32."""

    def __init__(self, layers: list[DeviceLayer], embedding: torch.Tensor, final_norm: torch.Tensor,
                 lm_head: tuple[torch.Tensor, object, int], pages: int, page: int = 64, max_tokens: int = 4096,
                 rope_theta: float = 10000.0):
        self.layers, self.embedding, self.final_norm = layers, embedding, final_norm
        self.head, t, self.vocab = lm_head
        if embedding.shape[0] < self.vocab:  # a chosen token is looked up there
            raise RuntimeError(f"Decoder: an embedding of {embedding.shape[0]} rows for a vocabulary of {self.vocab}")
        self.head_type = F.parse_type(t)
        first = layers[0]
        self.dev, self.cfg, self.page = first.dev, first.cfg, page
        self.max_tokens, self.max_pages = max_tokens, -(-max_tokens // page)
        dim = self.cfg.head_dim
        self.codes, self.scales = kv_pool(pages, len(layers), first.kv_heads, page, dim, device=self.dev)
        # build_rope_cache (vibeblade/transformer.py:102-112), float32 throughout; every position a row's
        # pages can hold
        inv = 1.0 / (rope_theta ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
        angle = torch.outer(torch.arange(self.max_pages * page, dtype=torch.float32), inv)
        self.cos, self.sin = angle.cos().to(self.dev), angle.sin().to(self.dev)

    def rows(self, n: int) -> Rows:
        """n empty rows over a pool with every page free."""
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=self.dev)  # noqa: E731
        return Rows(z(self.codes.shape[0]), z(n, self.max_pages) - 1, z(n), z(1))

    def _sent(self, values: list[int], dtype: torch.dtype = torch.int32) -> torch.Tensor:
        """A host list on the device, without waiting for it (a copy from pageable memory waits)."""
        t = torch.tensor(values, dtype=dtype)
        return t.pin_memory().to(self.dev, non_blocking=True) if self.dev.type == "cuda" else t

    def _rope(self, x: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
        """Rotate the halves of each head (vibeblade/transformer.py:73-99); at [T]: positions."""
        dim = self.cfg.head_dim
        x = x.view(x.shape[0], -1, dim)
        c, s = self.cos[at].unsqueeze(1), self.sin[at].unsqueeze(1)
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1).view(x.shape[0], -1)

    def forward(self, rows: Rows, tokens: torch.Tensor, new: list[int]) -> tuple[Rows, torch.Tensor]:
        """Append ``new[r]`` tokens to each row (``tokens`` [sum(new)], row after row) and run the
        blocks on them.  Returns the rows and the last block's output [sum(new), hidden].  Tokens past
        a row's pages count in ``missing`` and are not stored."""
        n = self._sent(new)
        q_start = torch.zeros(len(new) + 1, dtype=torch.int32, device=self.dev)
        torch.cumsum(n, 0, out=q_start[1:])
        refs, tables, lens, missing = kv_reserve(rows.refs, rows.tables, rows.lens, n, self.page)
        row = torch.repeat_interleave(torch.arange(len(new), device=self.dev), n, output_size=sum(new))
        at = rows.lens.long()[row] + torch.arange(sum(new), device=self.dev) - q_start.long()[row]
        at = at.clamp(max=self.cos.shape[0] - 1)  # past the row's pages there is no position
        x = self.embedding[tokens]
        prefill = x.shape[0] > DECODE_MAX_TOKENS
        for i, layer in enumerate(self.layers):
            def attention(q, k, v, i=i):
                q, k = self._rope(q, at), self._rope(k, at)
                kv_append(k, v, self.codes, self.scales, tables, lens, q_start, i)
                # a prompt's queries in bf16, as its matmuls take their inputs (the tcgen05 kernel)
                q = q.bfloat16() if prefill else q
                return kv_attention(q, self.codes, self.scales, tables, lens, q_start, i, max_new=max(new))
            x = layer.forward(x, attention)
        return Rows(refs, tables, lens, rows.missing + missing), x

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        """lm_head over the final norm of x [T, hidden] -> fp32 [T, vocab]."""
        h = rms_norm(x, self.final_norm, self.cfg.eps)
        return self.layers[0]._mm(h, self.head, self.cfg.hidden, self.vocab, self.head_type,
                                  prefill=x.shape[0] > DECODE_MAX_TOKENS)

    def score(self, prompts: list[list[int]]) -> list[torch.Tensor]:
        """Log probability of each prompt's tokens after its first, given those before."""
        new = [len(p) for p in prompts]
        self._fits(max(new, default=0))
        self._known(t for p in prompts for t in p)
        if sum(new) == 0:
            return [torch.empty(0, device=self.dev) for _ in prompts]
        tokens = self._sent([t for p in prompts for t in p], torch.long)
        rows, x = self.forward(self.rows(len(prompts)), tokens, new)
        self._have(rows)
        # row i predicts token i + 1; a prompt's last row has no token to score
        nxt = self._sent([t for p in prompts for t in (*p[1:], -1)])
        logprob = token_logprobs(self.logits(x), nxt)[0]
        return [lp[:-1] for lp in torch.split(logprob, new)]

    def beam_search(self, prompt: list[int], beams: int, steps: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The ``beams`` best continuations found of ``steps`` tokens: (tokens [beams, steps], their
        log probabilities [beams]), best first.  Up to 32 beams, and as many as the vocabulary has."""
        dev = self.dev
        if not 1 <= beams <= min(32, self.vocab):
            raise RuntimeError(f"Decoder: beams must be in 1..{min(32, self.vocab)}, got {beams}")
        if not prompt:
            raise RuntimeError("Decoder: the prompt is empty")
        self._known(prompt)
        self._fits(len(prompt) + max(steps - 1, 0))  # the last tokens are not run
        rows, x = self.forward(self.rows(1), self._sent(prompt, torch.long), [len(prompt)])
        logits = self.logits(x[-1:])
        total = torch.zeros(1, device=dev)
        out = torch.empty((1, 0), dtype=torch.int32, device=dev)
        for step in range(steps):
            _, _, lp, tok = token_logprobs(logits, None, beams)
            best, at = torch.topk((total[:, None] + lp).view(-1), beams)
            parents = (at // lp.shape[1]).to(torch.int32)
            total, chosen = best, tok.view(-1)[at]
            out = torch.cat([out[parents.long()], chosen[:, None]], dim=1)
            if step + 1 == steps:
                break
            refs, tables, lens, missing = kv_fork(self.codes, self.scales, rows.refs, rows.tables, rows.lens, parents)
            rows, x = self.forward(Rows(refs, tables, lens, rows.missing + missing), chosen.long(), [1] * beams)
            logits = self.logits(x)
        self._have(rows)
        return out, total

    def _fits(self, tokens: int) -> None:
        if tokens > self.max_tokens:
            raise RuntimeError(f"Decoder: a row of {tokens} tokens, max_tokens is {self.max_tokens}")

    def _known(self, tokens) -> None:
        for t in tokens:
            if not 0 <= t < self.embedding.shape[0]:
                raise RuntimeError(f"Decoder: token {t} is outside the vocabulary of {self.embedding.shape[0]}")

    def _have(self, rows: Rows) -> None:
        short = int(rows.missing.item())
        if short:
            raise RuntimeError(f"Decoder: the pool was {short} pages short")
