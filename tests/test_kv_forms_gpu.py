"""Forms of the KV cache's and the log probabilities' calls that long prompts, wide heads and tight masks
bring.  Tolerances as in tests/test_kv_gpu.py and tests/test_logprobs_gpu.py."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv_reference as R
import vibeblade_b200 as vb
from test_kv_gpu import DT, _attend, _state
from test_logprobs_gpu import check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (5, 1), (8, 1)])
@pytest.mark.parametrize("new,lens,window", [([70], [70], 0), ([33, 0, 129], [300, 12, 140], 0), ([90, 7], [250, 7], 31)])
def test_prompts_of_heads_of_256(cuda, dtype, heads, kv_heads, new, lens, window):
    _attend(cuda, lens, new, heads, kv_heads, 256, 32, dtype, window=window, seed=heads, max_new=max(new))
    _attend(cuda, lens, new, heads, kv_heads, 256, 16, dtype, window=window, seed=heads + 1, max_new=0)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_prompts_in_fp32(cuda, dim):
    _attend(cuda, [700, 430], [500, 430], 4, 2, dim, 64, torch.float32, seed=dim, max_new=500)


@pytest.mark.parametrize("lens,new,page,spare", [
    ([0], [131072], 16, 8200), ([100, 0, 33], [20000, 50000, 1], 32, 2400), ([17] * 5, [4000] * 5, 16, 1100),
])
def test_reserve_for_long_prompts(cuda, lens, new, page, spare):
    """Thousands of pages a row, and more than there are."""
    width = max((t + n) // page + 1 for t, n in zip(lens, new))
    pool, refs = _state(lens, page, dim=64, heads=1, layers=1, spare=spare, width=width)
    add = np.array(new, np.int32)
    got = vb.kv_reserve(*(torch.from_numpy(a).to(cuda) for a in (refs, pool.tables, pool.lens, add)), page)
    r, t, l, missing = R.reserve(refs, pool.tables, pool.lens, add, page)
    assert np.array_equal(got[0].cpu().numpy(), r) and np.array_equal(got[1].cpu().numpy(), t)
    assert np.array_equal(got[2].cpu().numpy(), l) and got[3].item() == missing


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows", [3, 520])
@pytest.mark.parametrize("left", [1, 3, 10])
def test_a_mask_that_leaves_few_tokens(cuda, dtype, rows, left):
    """Fewer tokens left than are listed, in one place or spread out: the list goes on with the masked
    ones in their order."""
    V = 20011
    for masked in (-math.inf, torch.finfo(dtype).min):
        x = logits(rows, V, left, dtype, cuda)
        keep = torch.zeros(rows, V, dtype=torch.bool, device=cuda)
        r = np.random.default_rng(left)
        for row in range(rows):
            keep[row, torch.from_numpy(r.choice(V, left, replace=False))] = True
        x = x.masked_fill(~keep, masked)
        t = keep.to(torch.int32).argmax(1).to(torch.int32)
        check(x, t, 20)


def test_scored_prompts_in_fp32(cuda):
    x = logits(700, 32001, 2, torch.float32, cuda)
    t = torch.from_numpy(np.random.default_rng(3).integers(0, 32001, 700).astype(np.int32)).to(cuda)
    check(x, t, 20)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_batch_of_both_kinds_sees_its_description_change(cuda, dim):
    """Lengths, tables and queries written in place before each call, with nothing waited for: the kernel
    for few rows starts beside the one for tiles and reads what was written before both."""
    new = [1, 150, 3, 1]
    states = [R.Pool(lens, 16, dim, 2, seed=9, spare=60, width=40) for lens in ([90, 300, 33, 1], [411, 160, 500, 77])]
    refs = []
    for i, pool in enumerate(states):
        q = torch.from_numpy(np.random.default_rng(i).normal(0, 1.5, (sum(new), 8 * dim)).astype(np.float32)).bfloat16().to(cuda)
        refs.append((q, *pool.on(cuda)))
    pages = min(r[1].shape[0] for r in refs)
    codes, scales = refs[1][1][:pages].contiguous(), refs[1][2][:pages].contiguous()
    for _, _, _, tables, _ in refs:
        tables.clamp_(max=pages - 1)
    qs = torch.from_numpy(R.q_start_of(new)).to(cuda)
    want = [vb.kv_attention(q, codes, scales, t, n, qs, max_new=150, with_lse=True) for q, _, _, t, n in refs]
    torch.cuda.synchronize()
    q, tables, lens = (torch.empty_like(refs[0][i]) for i in (0, 3, 4))
    got = []
    for i in range(60):
        q.copy_(refs[i % 2][0])
        tables.copy_(refs[i % 2][3])
        lens.copy_(refs[i % 2][4])
        got.append(vb.kv_attention(q, codes, scales, tables, lens, qs, max_new=150, with_lse=True))
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])
