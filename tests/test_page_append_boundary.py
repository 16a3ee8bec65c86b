"""PageAppend refuses what it cannot do before it launches anything: its plan takes pages and
moves the lengths, so a refusal after it would leave lengths over rows that were never written."""

import pytest

from test_paged_boundary import SLOTS, UNSUPPORTED, append, pool

from iron_b200.operators import PageAppend


@pytest.mark.parametrize("heads,dim", [(401, 128), (801, 64), (1024, 128)])
def test_rows_too_wide_for_summaries_are_refused_before_the_plan(heads, dim):
    # (without a GPU a launch would give a CUDA error instead)
    assert append(pool(kv_heads=heads, head_dim=dim, codes=4096, scales=4096)) == UNSUPPORTED
    with pytest.raises(ValueError, match="51200"):
        PageAppend(**(SLOTS | dict(num_kv_heads=heads, head_dim=dim, summaries=True)))
    PageAppend(**(SLOTS | dict(num_kv_heads=heads, head_dim=dim)))
    PageAppend(**(SLOTS | dict(num_kv_heads=51200 // dim, head_dim=dim, summaries=True)))
