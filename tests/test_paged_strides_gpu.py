"""Views whose dimensions of one element have odd strides."""

import random

import pytest
import torch

from paged_helpers import Cache, gen, randn, tree_reference
from test_page_select_gpu import call, check, summaries
from test_tree_attention_gpu import close, drafted, operator

pytestmark = pytest.mark.gpu


def odd(t):
    """The same values, with strides of 3 where there is one element."""
    return torch.as_strided(t, t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())])


@pytest.mark.parametrize("N,Hq,D", [(1, 1, 64), (5, 4, 64), (64, 4, 128)])
def test_tree_of_one_sequence_and_head(N, Hq, D):
    cache = Cache([300], 1, D, 64, 3, width=40)
    g = gen(3)
    q, kn, vn = randn(g, 1, N, Hq, D), randn(g, 1, N, 1, D), randn(g, 1, N, 1, D)
    parents = [drafted(random.Random(1), "random", N)]
    out = odd(torch.full_like(q, float("nan")))
    operator(cache, 1, N, Hq).get_callable()(odd(q), odd(kn), vn, cache.k, cache.v, cache.table, cache.lens,
                                             torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    close(out, *tree_reference(cache, q, kn, vn, parents, D**-0.5))


def test_selected_pages_of_one_sequence():
    cache = Cache([900], 1, 64, 32, 7)
    codes, scales = summaries(cache)
    q = randn(gen(7), 1, 1, 64)
    out, sel = call(cache, odd(q), codes, scales, 6, out=odd(torch.zeros_like(q)))
    check(cache, q, codes, scales, 6, out, sel)
