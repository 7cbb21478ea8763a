"""int32 and fp32 arrays of include/vbq_kv.h that are not aligned are refused on the host (a misaligned
address is a fault on the device)."""
from __future__ import annotations

import pytest

from vibeblade_b200 import _lib

N = 1 << 20  # workspace bytes, as many as are asked for


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, entry, args, at):
    """The call with the pointer `at` off by two bytes; nothing is launched."""
    bad = list(args)
    bad[at] += 2
    return getattr(lib, entry)(*bad) == _lib.VBQ_ERR_ALIGN and entry.encode() in lib.vbq_last_error()


#                refs tables lens new  pages page rows width refs' tables' lens' missing ws bytes stream
RESERVE = [16, 32, 48, 64, 100, 16, 7, 3, 16, 32, 48, 80, 16, N, None]
#       codes scales pages bytes scales page refs tables lens rows width parents rows' refs' tables' lens' missing ws
FORK = [16, 16, 100, 4096, 4, 16, 16, 32, 48, 7, 3, 64, 7, 16, 96, 112, 80, 16, N, None]
#          codes scales pages bytes scales page refs tables lens rows width refs' tables' live ws bytes stream
COMPACT = [16, 16, 100, 4096, 4, 16, 16, 32, 48, 7, 3, 16, 32, 80, 16, N, None]
#           x stride type rows vocab tokens top logprob entropy top_logprob top_token ws bytes stream
LOGPROBS = [16, 100, 0, 600, 100, 16, 3, 16, 16, 16, 16, None, 0, None]


@pytest.mark.parametrize("entry,args,pointers", [
    ("vbq_kv_reserve", RESERVE, (0, 1, 2, 3, 8, 9, 10, 11)), ("vbq_kv_fork", FORK, (1, 6, 7, 8, 11, 13, 14, 15, 16)),
    ("vbq_kv_compact", COMPACT, (1, 6, 7, 8, 11, 12, 13)), ("vbq_token_logprobs", LOGPROBS, (5, 7, 8, 9, 10)),
])
def test_misaligned_arrays(lib, entry, args, pointers):
    for at in pointers:
        assert refused(lib, entry, args, at), at
