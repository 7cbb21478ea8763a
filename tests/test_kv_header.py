"""What include/vbq_kv.h tells a C caller of the workspaces."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

HEADER = (Path(__file__).resolve().parents[1] / "include" / "vbq_kv.h").read_text()


@pytest.mark.parametrize("entry", ["vbq_kv_attention_workspace_bytes", "vbq_kv_pages_workspace_bytes",
                                   "vbq_token_logprobs_workspace_bytes"])
def test_every_workspace_says_what_has_to_be_zero(entry):
    comment = re.search(r"/\*((?:(?!\*/).)*)\*/\s*int " + entry, HEADER, re.S).group(1)
    assert "zero" in comment


def test_page_moves_name_the_pool():
    comment = re.search(r"/\*((?:(?!\*/).)*)\*/\s*int vbq_kv_pages_workspace_bytes", HEADER, re.S).group(1)
    assert "another number of pages" in " ".join(comment.replace("*", " ").split())
