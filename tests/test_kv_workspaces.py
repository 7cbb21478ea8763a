"""How much memory the KV cache's workspaces take."""
from __future__ import annotations

import ctypes as C

import pytest

from vibeblade_b200 import _lib


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_workspace_holds_what_the_grids_use(dim):
    """Two parts (O, the largest score, the sum) a CTA: of 16 rows for up to 4 CTAs an SM of the kernel for
    few rows, of 256 rows for one of the kernel for tiles, which takes dim 64 and 128; counters."""
    lib = _lib.load()
    v = C.c_size_t()
    _lib.check(lib.vbq_kv_attention_workspace_bytes(32, 8, dim, _lib.DTYPE_BF16, C.byref(v)), lib)
    parts = 4 * 2 * 148 * (4 * 16 * (dim + 2) + (256 * (dim + 2) if dim < 256 else 0))
    assert parts <= v.value <= parts + 16384
