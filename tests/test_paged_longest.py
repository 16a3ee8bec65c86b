"""Tables whose lengths, rounded up to whole tiles, would pass 32 bits are refused (without a
launch, so this runs without a GPU)."""

import pytest

from test_paged_boundary import POOL, SELECT, SHAPE, SLOTS, TREE, append, compact, fork, pool, select, tree

from iron_b200.operators import PageAppend, PageCompact, PageFork, PageSelectAttention, TreeAttention


@pytest.mark.parametrize("page", [16, 32, 64])
def test_a_length_rounds_up_within_32_bits(page):
    most = (1 << 31) // page - 1  # (2^31 - page) tokens: a tile of 64 or 128 more is past 2^31
    for entry in (tree, select, append, fork, compact):
        summaries = dict(codes=4096, scales=4096) if entry is select else {}
        assert entry(pool(page_size=page, max_pages=most, **summaries)) == SHAPE
    for cls, good in ((TreeAttention, TREE), (PageSelectAttention, SELECT), (PageAppend, SLOTS), (PageFork, SLOTS), (PageCompact, SLOTS)):
        with pytest.raises(ValueError, match="2\\^31 - 128"):
            cls(**(good | dict(page_size=page, max_pages=most)))
        cls(**(good | dict(page_size=page, max_pages=((1 << 31) - 128) // page)))


def test_the_tiles_of_a_batch_are_counted_within_32_bits():
    assert tree(pool(slots=1024, page_size=64, max_pages=1 << 21)) == SHAPE
    with pytest.raises(ValueError, match="batch"):
        TreeAttention(**(TREE | POOL | dict(batch=1024, page_size=64, max_pages=1 << 21)))
    TreeAttention(**(TREE | POOL | dict(batch=1000, page_size=64, max_pages=1 << 21)))
