"""What workspace a shared_prefix_attention call asks for."""

from __future__ import annotations

import pytest

KIB, PARTS = 1024, 256


def _size(rows, heads, batch, groups):
    from nanovllm_amd import _lib

    return _lib.lib.nvdsa_shared_prefix_attention_workspace_size(rows, heads, batch, groups)


def _sums(rows, heads):
    """Two sums a workgroup and pair of an item: 512 values and two more in fp32."""
    pairs = min(128, -(-rows * heads // 32) * 32)
    return 2 * PARTS * pairs * (2 * KIB + 8)


def _plan(rows, batch, groups):
    return 64 * (groups + batch) + 8 * rows + 32 * KIB


@pytest.mark.parametrize("rows,heads,batch", [(1, 16, 1), (64, 64, 64), (256, 128, 256), (16384, 16, 16384), (8192, 64, 8192)])
def test_calls_without_groups_have_no_room_for_shared_pairs(rows, heads, batch):
    """No pair has two items there: only what lies across parts is kept."""
    assert _sums(rows, heads) <= _size(rows, heads, batch, 0) <= _sums(rows, heads) + _plan(rows, batch, 0)


@pytest.mark.parametrize("rows,heads,batch,groups", [(64, 64, 64, 4), (5, 4, 2, 1), (4096, 16, 6, 2)])
def test_calls_with_groups_have_room_for_every_pair_twice(rows, heads, batch, groups):
    twice = 2 * min(rows * heads, 128 * batch) * (2 * KIB + 8)
    want = _sums(rows, heads) + twice
    assert want <= _size(rows, heads, batch, groups) <= want + _plan(rows, batch, groups)
