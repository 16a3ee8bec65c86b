"""Scores of 0 are equal whatever the sign of the zero: the lower page is kept."""

import pytest
import torch

from paged_helpers import Cache, gen, randn
from test_page_select_gpu import call, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_negative_zeros_tie_with_zeros(D):
    cache = Cache([50 * 16], 1, D, 16, 4)
    q = randn(gen(4), 1, 4, D).abs()
    codes = torch.randint(-127, -1, (cache.P, 1, 2, D), dtype=torch.int8, device="cuda")  # sums below 0 ...
    scales = torch.zeros(cache.P, 1, device="cuda")  # ... times 0
    codes[cache.table[0, 10:30].long()] = 0  # sums of 0
    out, sel = call(cache, q, codes, scales, 20)
    check(cache, q, codes, scales, 20, out, sel)
    assert sel[0, 0].tolist() == [*range(19), 49]
