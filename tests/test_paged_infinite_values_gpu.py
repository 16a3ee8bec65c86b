"""Cached values that are not finite: a row's output is the formula's softmax(..) V, infinite or
NaN in the column of such a value and as ever in the others. Probabilities enter the product with
V in two parts, and neither 0 nor a part of the other sign may meet an infinity."""

import math
import random

import pytest
import torch

from paged_helpers import Cache, attend, gen, randn, tree_reference
from test_page_select_gpu import call as select
from test_page_select_gpu import summaries
from test_tree_attention_gpu import drafted, operator

pytestmark = pytest.mark.gpu

INF = math.inf


def plant(cache):
    """Values of +inf, -inf, both, and NaN in some columns of every sequence with tokens."""
    for b, n in enumerate(cache.lens_list):
        if not n:
            continue
        at = lambda i: i % n  # noqa: E731
        for t, column, x in ((at(3), 1, INF), (at(n - 1), 2, -INF), (at(0), 5, INF), (at(n // 2 + 1), 5, -INF), (at(40), 7, math.nan)):
            if column == 5 and n == 1:
                continue
            page = int(cache.table[b, t // cache.page])
            cache.v[page, :, t % cache.page, column] = x
            cache.V[b][:, t, column] = x


def same(out, ref, tol):
    """Equal where the formula is not finite, within the tolerance elsewhere."""
    fine = torch.isfinite(ref)
    assert bool((torch.isnan(out) == torch.isnan(ref)).all())
    odd = ~fine & ~torch.isnan(ref)
    assert torch.equal(out.double()[odd], ref[odd]) and bool(odd.any())
    assert bool(((out.double() - ref).abs() <= tol)[fine].all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,Hq,width", [(2, 4, 40), (6, 4, 40), (8, 8, 900), (20, 8, 3000), (40, 8, 40), (128, 4, 40)])
def test_tree(D, N, Hq, width):
    cache = Cache([700, 0, 1, 64, 130, 2050], 2, D, 64, N, width=width)
    plant(cache)
    rng, g = random.Random(N), gen(N)
    q, kn, vn = randn(g, 6, N, Hq, D), randn(g, 6, N, 2, D), randn(g, 6, N, 2, D)
    parents = [drafted(rng, "ragged", N) for _ in range(6)]
    out = torch.empty_like(q)
    operator(cache, 6, N, Hq).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens,
                                             torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    ref, tol = tree_reference(cache, q, kn, vn, parents, D**-0.5)
    same(out, ref, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("copies", [1, 60])
def test_selected_pages(D, copies):
    """One CTA cluster per sequence and head, and (many sequences) pieces."""
    lens = [1, 700, 17, 2050, 0] * copies
    cache = Cache(lens, 2, D, 16, 3)
    codes, scales = summaries(cache)
    plant(cache)
    q = randn(gen(D), len(lens), 8, D)
    out, sel = select(cache, q, codes, scales, 200)  # every page
    refs = [attend(q[b].view(2, 4, D), cache.K[b], cache.V[b], D**-0.5) if n else (torch.zeros(2, 4, D, dtype=torch.float64, device="cuda"),) * 2
            for b, n in enumerate(lens)]
    same(out.view(len(lens), 2, 4, D), torch.stack([r[0] for r in refs]), torch.stack([r[1] for r in refs]))


def test_a_drafted_value_is_the_same_once_it_is_cached():
    """An infinite value of a node, and of the token that it becomes."""
    g = gen(4)
    for N, D in ((4, 64), (64, 128)):
        cache = Cache([100], 2, D, 64, 4)
        q, kn, vn = randn(g, 1, N, 8, D), randn(g, 1, N, 2, D), randn(g, 1, N, 2, D)
        cache.v[cache.table[0, 1].long(), :, 30, 9] = INF
        vn[0, 0, :, 11] = INF
        parents = torch.tensor([list(range(-1, N - 1))], dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)
        operator(cache, 1, N, 8).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, parents, out)
        assert bool((out[..., 9] == INF).all()) and bool((out[..., 11] == INF).all())
        out[..., 9] = out[..., 11] = 0
        assert bool(torch.isfinite(out).all())
