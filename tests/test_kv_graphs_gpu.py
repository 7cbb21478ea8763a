"""The KV cache's and the log probabilities' calls in CUDA graphs: what a graph holds stays its own
when later calls on its stream need more, and a graph may be the first to call."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as R
import vibeblade_b200 as vb
from test_kv_gpu import _q, _state

pytestmark = pytest.mark.gpu


def attention(cuda, lens, new, dim, seed, page=16, heads=8, kv_heads=2):
    """A call as a function of its output, on inputs of its own; lengths enough to need joins."""
    pool = R.Pool(lens, page, dim, kv_heads, seed=seed)
    q = _q(sum(new), heads * dim, seed, torch.bfloat16, cuda)[0]
    codes, scales, tables, ln = pool.on(cuda)
    qs = torch.from_numpy(R.q_start_of(new)).to(cuda)
    out = torch.empty_like(q)

    def call():
        vb.kv_attention(q, codes, scales, tables, ln, qs, max_new=max(new), out=out)
    return call, [out]


def logprobs(cuda, rows, vocab, top, seed):
    x = torch.from_numpy(np.random.default_rng(seed).normal(0, 3, (rows, vocab)).astype(np.float32)).to(cuda)
    t = torch.zeros(rows, dtype=torch.int32, device=cuda)
    outs = [torch.empty(rows, device=cuda), torch.empty(rows, device=cuda), torch.empty(rows, top, device=cuda),
            torch.empty(rows, top, dtype=torch.int32, device=cuda)]

    def call():
        for o, y in zip(outs, vb.token_logprobs(x, t, top)):
            o.copy_(y)
    return call, outs


def moves(cuda, rows, seed):
    """A fork, a reserve and a compaction; the pool's bytes are set back first, so that a replay repeats."""
    pool, refs = _state([37, 5, 64, 130], 16, spare=60, width=12, seed=seed)
    c0, s0, tables, ln = pool.on(cuda)
    codes, scales = c0.clone(), s0.clone()
    rf = torch.from_numpy(refs).to(cuda)
    parents = torch.tensor([(0, 0, 3, 1)[r % 4] if r < 8 else -1 for r in range(rows)], dtype=torch.int32, device=cuda)
    more = torch.ones(rows, dtype=torch.int32, device=cuda)
    outs = [torch.empty_like(rf), torch.empty(rows, 12, dtype=torch.int32, device=cuda),
            torch.empty(1, dtype=torch.int32, device=cuda), codes, scales]

    def call():
        codes.copy_(c0)
        scales.copy_(s0)
        r, t, n, _ = vb.kv_fork(codes, scales, rf, tables, ln, parents)
        r, t, n, _ = vb.kv_reserve(r, t, n, more, 16)
        for o, y in zip(outs, vb.kv_compact(codes, scales, r, t, n)):
            o.copy_(y)
    return call, outs


def store(cuda, n, seed):
    pool = R.Pool([100 + n, 30 + n], 16, 64, 2, seed=seed)
    c0, s0, tables, ln = pool.on(cuda)
    codes, scales = c0.clone(), s0.clone()
    qs = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=cuda)
    kv = _q(2 * n, 2 * 64, seed, torch.float32, cuda)[0]
    outs = [codes, scales, torch.empty_like(kv)]

    def call():
        codes.copy_(c0)
        scales.copy_(s0)
        vb.kv_append(kv, kv, codes, scales, tables, ln, qs)
        outs[2].copy_(vb.kv_read(codes, scales, tables, ln, qs, 2 * n)[0])
    return call, outs


CASES = {
    "attention": lambda cuda, big: attention(cuda, [3000, 2100], [1, 1], 128 if big else 64, 3 + big),
    "prompts": lambda cuda, big: attention(cuda, [2500, 300], [70, 200], 128 if big else 64, 5 + big),
    "logprobs": lambda cuda, big: logprobs(cuda, 8 if big else 1, 40000, 20 if big else 5, 7 + big),
    "moves": lambda cuda, big: moves(cuda, 300 if big else 8, 9 + big),
    "store": lambda cuda, big: store(cuda, 40 if big else 1, 11 + big),
}


def wanted(call, outs):
    """The outputs of a call on the current stream."""
    call()
    torch.cuda.synchronize()
    return [o.clone() for o in outs]


def blot(outs):
    for o in outs:
        o.fill_(77)


def same(outs, want):
    torch.cuda.synchronize()
    return all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("kind", CASES)
def test_a_larger_call_after_a_capture(cuda, kind):
    """The stream's later and larger calls leave a graph its workspace."""
    small, outs = CASES[kind](cuda, False)
    big, big_outs = CASES[kind](cuda, True)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        want = wanted(small, outs)
        with torch.cuda.graph(g, stream=st):
            small()
        big_want = wanted(big, big_outs)
        junk = [torch.full((n,), 77, dtype=torch.uint8, device=cuda) for n in (1 << 10, 1 << 16, 1 << 20, 1 << 24, 1 << 27)]
        for _ in range(3):
            blot(outs)
            g.replay()
            assert same(outs, want)
        blot(big_outs)
        big()
        assert same(big_outs, big_want)
        assert all((j == 77).all() for j in junk)


@pytest.mark.parametrize("kind", CASES)
def test_two_sizes_captured_on_one_stream(cuda, kind):
    calls = [CASES[kind](cuda, big) for big in (False, True)]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        wants = [wanted(*c) for c in calls]
        graphs = [torch.cuda.CUDAGraph() for _ in calls]
        for g, (call, _) in zip(graphs, calls):
            with torch.cuda.graph(g, stream=st):
                call()
        for i in (1, 0, 1, 0):
            blot(calls[i][1])
            graphs[i].replay()
            assert same(calls[i][1], wants[i])


@pytest.mark.parametrize("kind", CASES)
def test_a_capture_may_be_the_first_call(cuda, kind):
    """On a stream that has no workspaces: the graphs are replayed in another order than they were
    captured in, with calls on the stream itself between them."""
    calls = [CASES[kind](cuda, big) for big in (False, True, False)]
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        wants = [wanted(*c) for c in calls]
    st = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in calls]
    for g, (call, _) in zip(graphs, calls):
        with torch.cuda.graph(g, stream=st):
            call()
            call()  # shares the first's
    with torch.cuda.stream(st):
        for i in (2, 1):
            blot(calls[i][1])
            graphs[i].replay()
            assert same(calls[i][1], wants[i])
        blot(calls[0][1])
        calls[0][0]()  # eager, on the stream of the captures
        assert same(calls[0][1], wants[0])
        for i in (0, 2, 1, 0):
            blot(calls[i][1])
            graphs[i].replay()
            assert same(calls[i][1], wants[i])
