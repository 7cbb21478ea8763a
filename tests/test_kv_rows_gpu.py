"""Row tensors longer than the sequences' new tokens: a buffer of a fixed size whose q_start changes
on the device, as a captured step has it.  Tolerances as in tests/test_kv_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as R
import vibeblade_b200 as vb
from test_kv_gpu import DT, _check, _q

pytestmark = pytest.mark.gpu


def _longer(cuda, lens, new, rows, heads, kv_heads, dim, dtype, max_new, lead=0, page=16, seed=0):
    """out and lse of `rows` rows, the sequences' from row `lead` on, and the 64-bit form of theirs."""
    pool = R.Pool(lens, page, dim, kv_heads, seed=seed)
    q, q64 = _q(rows, heads * dim, seed, dtype, cuda)
    codes, scales, tables, ln = pool.on(cuda)
    qs = torch.from_numpy(R.q_start_of(new) + np.int32(lead)).to(cuda)
    wide = torch.full((rows, heads * dim + 64), 7.0, dtype=dtype, device=cuda)
    out, lse = vb.kv_attention(q, codes, scales, tables, ln, qs, out=wide[:, :heads * dim], max_new=max_new,
                               with_lse=True)
    n = sum(new)
    ref, ref_lse = R.attention(pool, q64[lead:lead + n], new, heads)
    assert (wide[:, heads * dim:] == 7).all()
    return out, lse, ref, ref_lse, 127 * float(pool.scales.max())


@pytest.mark.parametrize("hint", ["none", "rows", "right"])
@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(128, 8, 2, 64), (128, 32, 8, 64), (64, 16, 2, 200), (128, 4, 4, 300)])
@pytest.mark.parametrize("new", [1, 3, 10, 33])
def test_one_sequence_of_fewer_tokens_than_rows(cuda, dim, heads, kv_heads, rows, new, hint):
    out, lse, ref, ref_lse, vmax = _longer(cuda, [140 + new], [new], rows, heads, kv_heads, dim, torch.bfloat16,
                                           {"none": 0, "rows": rows, "right": new}[hint], seed=new)
    _check(out[:new].contiguous(), lse[:new], ref, ref_lse, vmax, torch.bfloat16)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new,lead,rows", [
    ([90, 5], [2, 1], 0, 9), ([90, 5], [2, 1], 3, 6), ([300, 90], [150, 40], 2, 260), ([300], [150], 0, 400),
    ([300], [0], 0, 200), ([40, 0], [0, 0], 0, 7), ([333, 50, 20], [1, 140, 1], 5, 147), ([30] * 40, [1] * 40, 1, 64),
])
def test_rows_of_no_sequence_see_nothing(cuda, dtype, dim, lens, new, lead, rows):
    out, lse, ref, ref_lse, vmax = _longer(cuda, lens, new, rows, 8, 2, dim, dtype, 0, lead=lead, seed=rows)
    n = sum(new)
    if n:
        _check(out[lead:lead + n].contiguous(), lse[lead:lead + n], ref, ref_lse, vmax, dtype)
    for part in (slice(0, lead), slice(lead + n, rows)):
        assert (out[part] == 0).all() and torch.isneginf(lse[part]).all()
