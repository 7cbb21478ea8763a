"""One workspace over calls of several sizes, through the C ABI and as its header allows."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

import kv_reference as R
from test_kv_gpu import _check, _q, _state
from test_logprobs_gpu import near, plain
from vibeblade_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib(cuda):
    return _lib.load()


def stream():
    return torch.cuda.current_stream().cuda_stream


def fork(lib, cuda, ws, lens, parents, spare):
    pool, refs = _state(lens, 16, spare=spare, seed=spare)
    codes, scales, tables, ln = pool.on(cuda)
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(cuda)  # noqa: E731
    rf, par, n = i(refs), i(parents), len(parents)
    width = pool.tables.shape[1]
    outs = [torch.full(s, 77, dtype=torch.int32, device=cuda) for s in ((pool.pages,), (n, width), (n,), (1,))]
    need = C.c_size_t()
    _lib.check(lib.vbq_kv_pages_workspace_bytes(pool.pages, max(n, len(lens)), C.byref(need)), lib)
    assert need.value <= ws.numel()
    _lib.check(lib.vbq_kv_fork(codes.data_ptr(), scales.data_ptr(), pool.pages, 2 * 2 * 2 * 16 * 64, 8, 16, rf.data_ptr(),
                               tables.data_ptr(), ln.data_ptr(), len(lens), width, par.data_ptr(), n,
                               *(o.data_ptr() for o in outs), ws.data_ptr(), ws.numel(), stream()), lib)
    c, s, r, t, l, missing = R.fork(pool.codes, pool.scales, refs, pool.tables, pool.lens, parents, 16)
    assert np.array_equal(outs[0].cpu().numpy(), r) and np.array_equal(outs[1].cpu().numpy(), t)
    assert np.array_equal(outs[2].cpu().numpy(), l) and outs[3].item() == missing
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)


def test_page_moves(cuda, lib):
    """Zeroed once a pool; within a pool any numbers of rows."""
    ws = torch.zeros(1 << 16, dtype=torch.uint8, device=cuda)
    for lens, parents, spare in (([37, 5, 64, 130], [0, 0, 3, 1], 9), ([300, 200], [0, 1, 0, 1] * 9, 40), ([1], [0, 0], 3)):
        ws.zero_()
        fork(lib, cuda, ws, lens, parents, spare)
        fork(lib, cuda, ws, lens, [0] * (3 * len(parents)), spare)
        fork(lib, cuda, ws, lens, [], spare)
        fork(lib, cuda, ws, lens, parents, spare)


def test_attention(cuda, lib):
    """Both kernels and every dim, only the first bytes zeroed."""
    need = C.c_size_t()
    most = 0
    for dim in (64, 128, 256):
        _lib.check(lib.vbq_kv_attention_workspace_bytes(8, 2, dim, 1, C.byref(need)), lib)
        most = max(most, need.value)
    ws = torch.full((most,), 0xa5, dtype=torch.uint8, device=cuda)
    ws[:16384] = 0
    for dim, new in ((64, [1, 1]), (128, [150, 1]), (256, [3, 1]), (64, [150, 70]), (128, [1, 1])):
        pool = R.Pool([1500, 900], 16, dim, 2, seed=dim)
        q, q64 = _q(sum(new), 8 * dim, dim, torch.bfloat16, cuda)
        codes, scales, tables, ln = pool.on(cuda)
        qs = torch.from_numpy(R.q_start_of(new)).to(cuda)
        out, lse = torch.empty_like(q), torch.empty(sum(new), 8, device=cuda)
        _lib.check(lib.vbq_kv_attention(q.data_ptr(), 8 * dim, out.data_ptr(), 8 * dim, lse.data_ptr(), 1, sum(new), 8,
                                        codes.data_ptr(), scales.data_ptr(), pool.pages, 1, 0, 2, 16, dim,
                                        tables.data_ptr(), tables.shape[1], ln.data_ptr(), qs.data_ptr(), 2,
                                        1 / math.sqrt(dim), 0, max(new), ws.data_ptr(), ws.numel(), stream()), lib)
        ref, ref_lse = R.attention(pool, q64, new, 8)
        _check(out, lse, ref, ref_lse, 127 * float(pool.scales.max()), torch.bfloat16)


def test_logprobs(cuda, lib):
    ws = torch.zeros(1 << 18, dtype=torch.uint8, device=cuda)
    for rows, vocab, top in ((1, 70000, 5), (8, 30000, 32), (2, 9000, 0), (300, 2500, 7), (1, 70000, 32)):
        x = torch.from_numpy(np.random.default_rng(rows).normal(0, 3, (rows, vocab)).astype(np.float32)).to(cuda)
        t = torch.zeros(rows, dtype=torch.int32, device=cuda)
        lp, en = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
        tl, ti = torch.empty(rows, top, device=cuda), torch.empty(rows, top, dtype=torch.int32, device=cuda)
        _lib.check(lib.vbq_token_logprobs(x.data_ptr(), vocab, 0, rows, vocab, t.data_ptr(), top, lp.data_ptr(),
                                          en.data_ptr(), tl.data_ptr(), ti.data_ptr(), ws.data_ptr(), ws.numel(), stream()), lib)
        ref = plain(x.double().cpu().numpy(), t.cpu().numpy(), top)
        for g, r in zip((lp, en, tl), ref):
            near(g, r)
        assert np.array_equal(ti.cpu().numpy(), ref[3])
