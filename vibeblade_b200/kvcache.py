"""The 8-bit paged KV cache, attention over it, moves of its pages, and log probabilities.

The steps around a block's matmuls that a decoding engine needs on the device (the reference
keeps fp32 keys and values and attends to them on the host, cpp/src/fast_model.cpp:690-804):

    codes, scales = kv_pool(pages, layers, kv_heads, page, dim)
    refs, tables, lens, missing = kv_reserve(refs, tables, lens, new_tokens, page)
    kv_append(k, v, codes, scales, tables, lens, q_start, layer)       # per layer, after RoPE
    attn = kv_attention(q, codes, scales, tables, lens, q_start, layer)
    logprob, entropy, top_logprob, top_token = token_logprobs(logits, tokens, top)
    refs, tables, lens, missing = kv_fork(codes, scales, refs, tables, lens, parents)

``codes`` is int8 [pages, layers, 2, kv_heads, page, dim] and ``scales`` fp32 [pages, layers, 2,
kv_heads]: a stored value is scale * code, one scale a page, layer, head and K / V.  Sequences
are rows of ``tables`` (int32 [seqs, max_pages], page numbers, -1 for none) with ``lens`` tokens
(int32 [seqs], new ones included); ``q_start`` (int32 [seqs + 1]) says which rows of q, k and v
are each sequence's last tokens.  ``refs`` (int32 [pages]) counts the rows that hold a page; 0
is free.  Everything stays on the device: no call synchronises, and each may be captured in a
CUDA graph.  Calls share workspaces by stream, which are made by the first call that needs them and
kept; graphs captured on one stream after such a call share them too, so they are replayed one after
the other.  A call captured before that has a workspace in its graph's own pool, cleared at each replay.
"""
from __future__ import annotations

import torch

from . import _lib

_F = None  # the extension of face/kv_face.cpp: the calls' checks, allocations and C entries


def _load():
    """Loads the extension on the first call (there is no fallback: without it every call raises)."""
    global _F
    _lib.load()
    try:
        from . import _kvface
    except ImportError as e:
        raise RuntimeError("_kvface.so not found or not loadable: build it with `python -m vibeblade_b200.build` "
                           f"({e})") from e
    _F = _kvface
    return _F


def kv_pool(pages: int, layers: int, kv_heads: int, page: int, dim: int,
            device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An empty pool: (codes, scales).  ``page`` is 16, 32, 64 or 128 tokens, ``dim`` 64, 128 or 256."""
    if page not in (16, 32, 64, 128):
        raise RuntimeError("kv_pool: " + f"page must be 16, 32, 64 or 128 tokens, got {page}")
    if dim not in (64, 128, 256):
        raise RuntimeError("kv_pool: " + f"dim must be 64, 128 or 256, got {dim}")
    if min(pages, layers, kv_heads) < 1:
        raise RuntimeError("kv_pool: " + "pages, layers and kv_heads must be at least 1")
    return (torch.zeros((pages, layers, 2, kv_heads, page, dim), dtype=torch.int8, device=device),
            torch.zeros((pages, layers, 2, kv_heads), dtype=torch.float32, device=device))


def kv_append(k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
              tables: torch.Tensor, lens: torch.Tensor, q_start: torch.Tensor, layer: int = 0) -> None:
    """Quantise the batch's new keys and values ([rows, kv_heads * dim], fp32 or bf16; columns
    of a packed matmul output are taken as they are) into layer ``layer`` of the pool.  A page's
    scale grows to the largest new value / 127 and its earlier codes are rescaled with it; see
    vbq_kv_append for the rounding."""
    (_F or _load()).append(k, v, codes, scales, tables, lens, q_start, layer)


def kv_read(codes: torch.Tensor, scales: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
            q_start: torch.Tensor, rows: int, layer: int = 0,
            dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that layer ``layer`` holds for the batch's rows (q_start's, ``rows``
    of them: each sequence's last tokens): two [rows, kv_heads * dim] tensors."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError("kv_read: dtype must be torch.float32 or torch.bfloat16")
    return (_F or _load()).read(codes, scales, tables, lens, q_start, rows, layer, dtype is torch.bfloat16)


def kv_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, tables: torch.Tensor,
                 lens: torch.Tensor, q_start: torch.Tensor, layer: int = 0, *, scale: float | None = None,
                 window: int = 0, max_new: int = 0, out: torch.Tensor | None = None, with_lse: bool = False):
    """Causal attention of the batch's rows (q [rows, heads * dim], fp32 or bf16) over layer
    ``layer`` of the pool, the rows' own keys and values appended before.  Row i of a
    sequence's n new tokens sees the tokens up to its own, the last ``window`` of them if that
    is not 0.  ``scale`` defaults to dim ** -0.5.  ``max_new``: the most new tokens a sequence
    has, where known (it selects the kernel).  Returns out [rows, heads * dim], with
    ``with_lse`` also the fp32 [rows, heads] log-sum-exp.  A row that sees nothing, or
    that no sequence has (before q_start's first and from its last on), gives zeros and -inf."""
    return (_F or _load()).attention(q, codes, scales, tables, lens, q_start, layer, scale, window, max_new, out,
                                     bool(with_lse))


def kv_reserve(refs: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, new_tokens: torch.Tensor, page: int):
    """Pages for ``new_tokens`` (int32 [rows]) more tokens a row, the lowest free ones first:
    new (refs, tables, lens, missing), ``missing`` an int32 [1] count of pages there were not."""
    return (_F or _load()).reserve(refs, tables, lens, new_tokens, page)


def kv_fork(codes: torch.Tensor, scales: torch.Tensor, refs: torch.Tensor, tables: torch.Tensor,
            lens: torch.Tensor, parents: torch.Tensor):
    """Regroup sequences: new row r continues row ``parents[r]`` (int32; -1: an empty row).
    Whole pages are shared, a part-filled last page is copied for every row after the first
    that continues it, rows nobody continues are freed.  Copies, forks, reorders and frees are
    all this call.  Returns new (refs, tables, lens, missing)."""
    return (_F or _load()).fork(codes, scales, refs, tables, lens, parents)


def kv_compact(codes: torch.Tensor, scales: torch.Tensor, refs: torch.Tensor, tables: torch.Tensor,
               lens: torch.Tensor):
    """Make the pool dense: pages in use move down into the free ones below, in order.
    Returns new (refs, tables, live), ``live`` an int32 [1] count of pages in use, which then
    are 0 .. live - 1."""
    return (_F or _load()).compact(codes, scales, refs, tables, lens)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top: int = 0):
    """(logprob [rows], entropy [rows], top_logprob [rows, top], top_token int32 [rows, top]) of
    logits [rows, vocab] (fp32 or bf16, columns adjacent): the log probability of the given
    tokens (int32 [rows]; one outside the vocabulary has 0; None when ``tokens`` is), the
    entropy in nats, and the ``top`` (0 .. 32) likeliest tokens in descending order, equal ones
    by the lower token."""
    return (_F or _load()).logprobs(logits, tokens, top)
