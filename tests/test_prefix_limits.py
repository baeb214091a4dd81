"""What `b200q_prefix_attention` takes, by the size of its scratch memory: arithmetic of the host."""

from __future__ import annotations

import pytest

from linnet_b200 import _lib


def scratch(batch, nq, nkv, head_dim, prefix, max_seq):
    return _lib.load().b200q_prefix_attention_scratch_bytes(batch, nq, nkv, head_dim, prefix, max_seq)


@pytest.mark.parametrize("shape", [
    (65537, 8, 8, 64, 0, 1), (1, 8, 3, 64, 0, 1), (1, 129, 1, 64, 0, 1), (1, 8, 8, 96, 0, 1), (1, 0, 0, 64, 0, 1), (-1, 8, 8, 64, 0, 1),
    (1, 8, 8, 64, -1, 1), (1, 8, 8, 64, 1 << 30, 1), (1, 8, 8, 64, 0, 1 << 30), (65536, 65536, 65536, 64, 0, 0),
    (1, 8, 8, 128, (1 << 30) - 1, 1),  # 2 * 8 * 2^24 tiles: 2 TB a tensor
    # a prefix of 2^20 keys for 65536 rows of 8 heads: 2^28 tiles of 128 rows, seconds on every multiprocessor
    (65536, 32, 8, 128, 1 << 20, 0), (65536, 64, 64, 64, 0, 2048)])
def test_shapes_that_are_not_taken(shape):
    assert scratch(*shape) == -1 and "prefix_attention" in _lib.last_error()


@pytest.mark.parametrize("batch,nq,nkv,head_dim,prefix,max_seq", [
    (0, 8, 8, 64, 100, 10), (1, 1, 1, 64, 0, 0), (1, 1, 1, 128, (1 << 30) - 1, 1), (64, 32, 8, 128, 8192, 512), (65536, 32, 8, 128, 8192, 64),
    (65536, 300, 300, 64, 0, 1)])
def test_scratch_holds_a_part_of_every_item_and_block(batch, nq, nkv, head_dim, prefix, max_seq):
    """Of every row's own keys and head (and of one more for every block) a part of rep rows of D sums, a
    maximum and a sum; of the prefix two of 128 rows for every item; whole 16-byte steps."""
    size, rep = scratch(batch, nq, nkv, head_dim, prefix, max_seq), nq // nkv
    items = nkv * -(-batch // (2 * (128 // rep))) if prefix else 0
    least = 4 * (batch * nkv * rep * (head_dim + 2) + items * 2 * 128 * (head_dim + 2))
    assert size % 16 == 0 and size >= least
    assert size <= least + 4 * (batch * nkv * 3 + 148 * (2 * 128 + rep) * (head_dim + 2) + 148 * 3 + batch + 8)
