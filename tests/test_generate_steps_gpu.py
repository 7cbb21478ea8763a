"""A step of the serving loop does not wait for the device."""
from __future__ import annotations

import pytest
import torch

import vibeblade_b200 as vb
from test_generate_gpu import decoder, prompt  # noqa: F401  (decoder is the fixture)

pytestmark = pytest.mark.gpu


def test_steps_do_not_synchronise(decoder):  # noqa: F811
    """A prompt, a fork into three rows and a token for each."""
    p = torch.tensor(prompt(20, 3), device=decoder.dev)
    parents = torch.zeros(3, dtype=torch.int32, device=decoder.dev)

    def steps():
        rows, x = decoder.forward(decoder.rows(1), p, [20])
        _, _, _, tok = vb.token_logprobs(decoder.logits(x[-1:]), None, 3)
        refs, tables, lens, missing = vb.kv_fork(decoder.codes, decoder.scales, rows.refs, rows.tables, rows.lens, parents)
        return decoder.forward(type(rows)(refs, tables, lens, missing), tok.view(-1).long(), [1, 1, 1])[1]

    first = steps()  # workspaces are made
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        again = steps()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(first, again)
