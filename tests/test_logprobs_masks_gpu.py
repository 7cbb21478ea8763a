"""Log probabilities of rows whose largest logit is the type's lowest value, with -inf beside it, and
of logits near the ends of fp32.  Tolerances as in tests/test_logprobs_gpu.py (x - max is exact or
vanishes here)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import vibeblade_b200 as vb
from test_logprobs_gpu import DT, near, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,V", [(1, 4), (3, 41), (2, 5000), (1, 70000), (700, 3001)])
@pytest.mark.parametrize("off", [0, 1, 5])
def test_infinities_beside_the_lowest_value(cuda, dtype, rows, V, off):
    """Every second, and every but the seventh, logit -inf, the others the type's lowest value: the row
    is uniform over those, wherever it begins in memory."""
    low = torch.finfo(dtype).min
    for step in (2, 7):
        big = torch.full((rows, V + 8), -math.inf, dtype=dtype, device=cuda)
        x = big[:, off:off + V]
        x[:, ::step] = low
        n = len(range(0, V, step))
        top = min(32, n)
        t = torch.tensor([r % 2 for r in range(rows)], dtype=torch.int32, device=cuda)
        lp, en, tl, ti = vb.token_logprobs(x, t, top)
        near(lp, np.where(np.arange(rows) % 2 == 0, -math.log(n), -math.inf))
        near(en, np.full(rows, math.log(n)))
        near(tl, np.full((rows, top), -math.log(n)))
        assert torch.equal(ti.cpu(), torch.arange(0, step * top, step, dtype=torch.int32).expand(rows, top))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows", [2, 600])
def test_lowest_values_in_one_part_of_a_row(cuda, dtype, rows):
    """-inf and the lowest value together where the row's largest logit is an ordinary one, or NaN."""
    V, low = 9000, torch.finfo(dtype).min
    x = torch.full((rows, V), -math.inf, dtype=dtype, device=cuda)
    x[:, ::3] = low
    x[1, 8000:8003] = torch.tensor([1.0, 2.0, 1.0], device=cuda).to(dtype)
    t = torch.full((rows,), 8001, dtype=torch.int32, device=cuda)
    got = vb.token_logprobs(x, t, 3)
    ref = plain(x[1:2].double().cpu().numpy(), [8001], 3)
    for g, r in zip((got[0], got[1], got[2]), ref):
        near(g[1:2], r)
    assert got[3][1].tolist() == [8001, 8000, 8002]
    near(got[1][:1], [math.log(V / 3)])
    x[0, 5] = math.nan
    got = vb.token_logprobs(x, t, 3)
    assert torch.isnan(got[0][0]) and torch.isnan(got[1][0])


@pytest.mark.parametrize("rows", [1, 600])
def test_logits_at_both_ends_of_fp32(cuda, rows):
    """Differences past fp32's range are weights of zero, in the entropy too."""
    x = torch.full((rows, 4101), -3e38, device=cuda)
    x[:, 17] = 3e38
    x[:, 4100] = 3e38
    t = torch.full((rows,), 17, dtype=torch.int32, device=cuda)
    lp, en, tl, ti = vb.token_logprobs(x, t, 2)
    near(lp, np.full(rows, -math.log(2)))
    near(en, np.full(rows, math.log(2)))
    near(tl, np.full((rows, 2), -math.log(2)))
    assert ti[0].tolist() == [17, 4100]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows", [2, 600])
@pytest.mark.parametrize("off", [0, 3])
def test_lists_that_overflow(cuda, dtype, rows, off):
    """More elements reach the list's bound than it holds: large logits crowded into the vectors of a few
    threads, in falling and in rising order, beside ties, and ties at the row's end."""
    V = 40003
    r = np.random.default_rng(rows + off)
    big = torch.from_numpy(r.normal(0, 1, (rows, V + 8)).astype(np.float32)).to(dtype).to(cuda)
    x = big[:, off:off + V]
    at = torch.arange(V, device=cuda) + off
    per = 512 if rows > 512 else 256
    lanes = (at // (8 if dtype == torch.bfloat16 else 4)) % per < 6  # of six threads, or about
    n = int(lanes.sum())
    steps = torch.arange(n, device=cuda, dtype=torch.float32)
    for edit in range(5):
        y = x.clone()
        if edit == 0:
            y[:, lanes] = (100 + steps / 16).to(dtype)
        elif edit == 1:
            y[:, lanes] = (100 - steps / 16).to(dtype)
        elif edit == 2:
            y[:, lanes] = (100 + (steps * 7919 % 97)).to(dtype)
        elif edit == 3:
            y[:] = -math.inf
            y[:, -40:] = 1.0
            y[:, 100] = 2.0
        else:
            y[:] = -math.inf
            y[:, 7] = 3.0
            y[:, -5:] = torch.tensor([1.0, 2.0, 1.0, 2.0, 1.0], device=cuda).to(dtype)
            y[:, 9000] = math.nan
        if edit == 4:  # a NaN spoils the sums, not the list
            ti = vb.token_logprobs(y, None, 9)[3]
            want = [7, V - 4, V - 2, V - 5, V - 3, V - 1, 0, 1, 2]
            assert (ti.cpu() == torch.tensor(want, dtype=torch.int32)).all()
            continue
        for top in (1, 20, 32):
            got = vb.token_logprobs(y, None, top)
            _, en, tl, ti = plain(y[:2].double().cpu().numpy(), None, top)
            assert np.array_equal(got[3][:2].cpu().numpy(), ti)
            near(got[2][:2], tl)
            near(got[1][:2], en)
