"""Attention over values and queries at the ends of their ranges, and over long caches.  Tolerances as
in tests/test_kv_gpu.py."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv_reference as R
import vibeblade_b200 as vb
from test_kv_gpu import DT, _attend, _check, _q

pytestmark = pytest.mark.gpu


def _two_scores(cuda, dtype, new, dim, values, L=40960):
    """8 KV heads of 8 query heads over L tokens, of which the first 128 score 0 and the others
    7.8 log 2: (out, lse, the second score, codes, scales)."""
    kv, group, page = 8, 8, 128
    n = L // page
    g = torch.Generator(device=cuda).manual_seed(dim)
    codes = torch.zeros((n, 1, 2, kv, page, dim), dtype=torch.int8, device=cuda)
    scales = torch.zeros((n, 1, 2, kv), device=cuda)
    codes[1:, :, 0] = 127
    scale = dim ** -0.5
    ks = float(np.float32(7.8 * math.log(2) / (127 * dim * scale)))
    scales[1:, :, 0] = ks
    if values:
        codes[:, :, 1] = torch.randint(-127, 128, codes[:, :, 1].shape, generator=g, dtype=torch.int8, device=cuda)
        scales[:, :, 1] = 0.005 + 0.02 * torch.rand(scales[:, :, 1].shape, generator=g, device=cuda)
    q = torch.ones(new, kv * group * dim, dtype=dtype, device=cuda)
    tables = torch.arange(n, dtype=torch.int32, device=cuda)[None].contiguous()
    out, lse = vb.kv_attention(q, codes, scales, tables, torch.tensor([L], dtype=torch.int32, device=cuda),
                               torch.tensor([0, new], dtype=torch.int32, device=cuda), max_new=new, with_lse=True)
    s = 127 * dim * ks * scale
    seen = L - new + np.arange(new) + 1
    ref_lse = np.log(page + (seen - page) * math.exp(s))
    assert np.abs(lse.double().cpu().numpy() - ref_lse[:, None]).max() <= 2e-5 + 2.0 ** -22 * ref_lse.max()
    return out, s, codes, scales


@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, 600), (torch.bfloat16, 1), (torch.float32, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_caches_of_equal_scores(cuda, dtype, new, dim):
    """Tens of thousands of equal weights: their sum's roundings go one way."""
    out, s, codes, scales = _two_scores(cuda, dtype, new, dim, True)
    page, kv, L = 128, 8, 40960
    v = (codes[:, 0, 1].double() * scales[:, 0, 1].double()[..., None, None]).permute(0, 2, 1, 3).reshape(L, kv, dim)
    v[page:] *= math.exp(s)
    seen = L - new + torch.arange(new, device=cuda)
    z = page + (seen + 1 - page).double() * math.exp(s)
    ref = v.cumsum(0)[seen] / z[:, None, None]
    err = (out.double().view(new, kv, 8, dim) - ref[:, :, None]).abs()
    vmax = 127 * float(scales.max())
    if dtype == torch.float32:
        assert err.max() <= 2e-5 * vmax
    else:
        assert (err <= 2.0 ** -10 * vmax + 2.0 ** -8 * ref[:, :, None].abs()).all()


@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, 600), (torch.bfloat16, 1), (torch.float32, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_caches_of_zero_values(cuda, dtype, new, dim):
    """Blocks of zeros have the scale 0; the sum of exponentials over them stays in range when the later
    scores lie 2^7.8 above the first ones', which a lazily moved reference lets pass."""
    out = _two_scores(cuda, dtype, new, dim, False)[0]
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_infinite_queries_give_nan_in_their_rows(cuda, dtype, new, value):
    """Scores of +-inf or NaN have no softmax: the row is NaN, whatever the sign of the keys' codes."""
    pool = R.Pool([260], 32, 128, 2, seed=8)
    pool.codes[:, :, 0, :, :, 3] = -5  # one sign for every key
    q, q64 = _q(new, 4 * 128, 1, dtype, cuda)
    q[0, 3] = value
    q64[0, :128] = 0
    codes, scales, tables, ln = pool.on(cuda)
    out, lse = vb.kv_attention(q, codes, scales, tables, ln, torch.tensor([0, new], dtype=torch.int32, device=cuda),
                               with_lse=True, max_new=new)
    assert torch.isnan(out[0, :128]).all() and torch.isnan(lse[0, 0])
    ref, ref_lse = R.attention(pool, q64, [new], 4)
    out[0, :128] = torch.from_numpy(ref[0, 0]).to(out)
    lse[0, 0] = float(ref_lse[0, 0])
    _check(out, lse, ref, ref_lse, 127 * float(pool.scales.max()), dtype)


@pytest.mark.parametrize("dim", [64, 128])
def test_half_a_million_equal_scores(cuda, dim):
    """The sum's roundings do not grow with the cache."""
    _two_scores(cuda, torch.bfloat16, 600, dim, True, L=524288)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 1 << 30])
def test_the_largest_windows(cuda, dtype, dim, window):
    """Beside rows before a sequence's first token, from whose places they would reach past int32."""
    for lens, new in (([22, 0, 9, 3], [30, 12, 9, 10]), ([10, 40], [150, 170]), ([200], [230])):
        _attend(cuda, lens, new, 8, 2, dim, 16, dtype, window=window, seed=dim)
