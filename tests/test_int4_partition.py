"""Split counts of the 4-bit history branch (no GPU)."""

import pytest

from oscar_new_amd.config import (INT4_SLOTS, SPLIT_ROW_BYTES, choose_device_partition,
                                  choose_int4_splits)


@pytest.mark.parametrize("tokens", [17, 64, 300, 2048, 16384])
@pytest.mark.parametrize("requests,kv_heads,heads", [(1, 1, 6), (8, 2, 12), (64, 4, 4)])
def test_splits_of_row_tiles(tokens, requests, kv_heads, heads):
    assert choose_int4_splits(tokens, requests, kv_heads, heads, None) == 1
    assert choose_int4_splits(tokens, requests, kv_heads, heads, 0) == 1
    before = 1
    for longest in (1, 256, 1000, 8000, 131072):
        splits = choose_int4_splits(tokens, requests, kv_heads, heads, longest)
        assert 1 <= splits <= min(16, -(-longest // 256))
        assert splits * tokens * heads * SPLIT_ROW_BYTES <= 128 << 20 or splits == 1
        assert splits >= before or tokens * heads > 256 * 32  # few tiles: longer histories split more
        before = splits


def test_a_tile_for_every_unit_is_not_split():
    # 256 tiles of 32 rows are a workgroup per CU already; half of them leave room for two splits.
    assert choose_int4_splits(8192, 1, 1, 1, 32768) == 1
    assert choose_int4_splits(4096, 1, 1, 1, 32768) == 2


def test_slots_of_the_device_rule():
    splits, share = choose_device_partition(32, 1, 1, 32, 6, slots=INT4_SLOTS)
    assert share == -INT4_SLOTS and splits >= INT4_SLOTS // 32
    assert choose_device_partition(32, 1, 1, 32, 6)[1] == -512  # the 2-bit kernels' own
    assert choose_device_partition(32, 1, 17, 32, 6, slots=INT4_SLOTS) == (1, 0)
