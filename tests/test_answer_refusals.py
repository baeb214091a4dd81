"""Calls of the operators for many answers to one prompt that are refused before anything is allocated or
launched."""

from __future__ import annotations

import pytest
import torch

from linnet_b200 import glue


@pytest.mark.gpu
@pytest.mark.parametrize("top", [-1, 33, 1 << 45, 8])
def test_alternatives_that_there_are_none_of(top):
    """An absurd number is no question of memory; more than the row has are refused too."""
    logits = torch.zeros(2, 7 if top == 8 else 1000, device="cuda")
    tokens = torch.zeros(2, dtype=torch.long, device="cuda")
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    with pytest.raises(ValueError, match="alternatives of a row"):
        glue.token_logprobs(logits, tokens, top)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
