"""The GEMV calls' split-K scratch, by stream."""
from __future__ import annotations

import weakref

import pytest
import torch

from vibeblade_b200 import dequant


@pytest.fixture(autouse=True)
def own_scratch(monkeypatch):
    monkeypatch.setattr(dequant, "_SCRATCH", {})


def test_a_buffer_that_was_handed_out_stays():
    """A captured graph may hold its address, so a larger call's buffer does not free it."""
    dev = torch.device("cpu", 0)
    first = weakref.ref(dequant._stream_scratch(dev, 7, 100))
    assert first().numel() >= 100 and not first().any()
    assert dequant._stream_scratch(dev, 7, 50) is first()
    second = dequant._stream_scratch(dev, 7, first().numel() + 1)
    assert first() is not None and second is not first() and not second.any()
    assert dequant._stream_scratch(dev, 7, 100) is second
    assert dequant._stream_scratch(dev, 8, 100) is not second
