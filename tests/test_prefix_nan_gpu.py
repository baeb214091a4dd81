"""`glue.prefix_attention` of rows whose every score is NaN: the row is NaN, and no other is.

Lengths are whole tiles of 64 keys, so that no masked key stands beside the NaN scores, and both forms
of the joining kernel are met (few parts a row, and many)."""

from __future__ import annotations

import math

import pytest
import torch

from linnet_b200 import glue
from tests.test_prefix_attention_gpu import _inputs, _no_wait_expired, _want  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [  # batch, nq, nkv, hd, prefix, slots
    (3, 4, 2, 64, 128, 0), (5, 8, 2, 128, 128, 64), (40, 32, 8, 128, 256, 128), (300, 8, 2, 64, 192, 64), (7, 4, 1, 128, 0, 64),
    (2, 4, 2, 64, 64 * 640, 0), (2, 4, 2, 128, 64 * 640, 128), (70, 4, 1, 64, 64 * 300, 64)]


def _check(args, wrong):
    """`wrong` [batch, nq]: the heads that are NaN."""
    got = glue.prefix_attention(*args).view(args[0].shape)
    assert torch.equal(got.isnan().all(dim=-1), wrong) and torch.equal(got.isnan().any(dim=-1), wrong)
    q = args[0].nan_to_num()
    want, allowed = _want(q, args[1].nan_to_num(), *args[2:])
    right = ~wrong[:, :, None].expand_as(got)
    over = ((got.double() - want.view(got.shape)).abs() / allowed.view(got.shape))[right]
    assert over.numel() == 0 or over.max().item() <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_query_that_is_nan(shape, dtype):
    args = _inputs(*shape, dtype)
    q, positions = args[0], args[-1]
    positions.fill_(shape[-1] - 1)
    wrong = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    wrong[1, 2] = wrong[-1, 0] = True
    q[wrong] = math.nan
    _check(args, wrong)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[4]], ids=str)
def test_a_prompt_that_is_nan(shape):
    """The keys of one KV head, whole: its heads are NaN whatever else they see."""
    args = _inputs(*shape, torch.bfloat16)
    q, pk, positions = args[0], args[1], args[-1]
    positions.fill_(shape[-1] - 1)
    heads, kv_heads = shape[1], shape[2]
    pk[-1] = math.nan
    wrong = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    wrong[:, heads - heads // kv_heads:] = True
    _check(args, wrong)
