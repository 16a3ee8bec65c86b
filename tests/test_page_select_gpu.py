"""PageSelectAttention against the rule: the selected pages are equal, the outputs within
the derived tolerance of paged_helpers.attend of float64."""

import math
import random

import pytest
import torch

from paged_helpers import Cache, attend, gen, randn, select_reference, summary

pytestmark = pytest.mark.gpu

from iron_b200.operators import PageSelectAttention


def summaries(cache):
    """Codes and scales of the pages in use; garbage elsewhere, and for partial pages."""
    codes = torch.randint(-128, 128, (cache.P, cache.Hkv, 2, cache.D), dtype=torch.int8, device="cuda")
    scales = torch.full((cache.P, cache.Hkv), math.nan, device="cuda")
    for s, n in enumerate(cache.lens_list):
        ids = cache.table[s, : n // cache.page].long()
        if len(ids):
            c, x = summary(cache.k[ids])
            codes[ids], scales[ids] = c.to("cuda", torch.int8), x.cuda()
    return codes, scales


def call(cache, q, codes, scales, top, out=None):
    B, Hq, D = q.shape
    op = PageSelectAttention(batch=B, num_heads=Hq, num_kv_heads=cache.Hkv, head_dim=D, page_size=cache.page, num_pages=cache.P,
                             max_pages=cache.M, top_pages=top)
    out = torch.full((B, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda") if out is None else out
    sel = torch.full((B, cache.Hkv, top), -9, dtype=torch.int32, device="cuda")
    op.get_callable()(q, cache.k, cache.v, codes, scales, cache.table, cache.lens, out, sel)
    return out, sel


def check(cache, q, codes, scales, top, out, sel, values=True):
    B, Hq, D = q.shape
    g = Hq // cache.Hkv
    for b, L in enumerate(cache.lens_list):
        n = -(-L // cache.page)
        ids = cache.table[b, :n].long()
        for h in range(cache.Hkv):
            x = q[b, h * g : h * g + g]
            keep = select_reference(x, codes[ids, h], scales[ids, h], top)
            assert sel[b, h].tolist() == keep + [-1] * (top - len(keep)), (b, h)
            o = out[b, h * g : h * g + g].double()
            if not keep:
                assert not bool(o.any())
            elif values:
                t = torch.cat([torch.arange(i * cache.page, min(L, (i + 1) * cache.page)) for i in keep]).cuda()
                ref, tol = attend(x, cache.K[b][h, t], cache.V[b][h, t], 1 / math.sqrt(D))
                assert bool(((o - ref).abs() <= tol).all()), (b, h)


def run(lens, top, Hq, Hkv, D, page, seed=0, width=None):
    cache = Cache(lens, Hkv, D, page, seed, width=width)
    codes, scales = summaries(cache)
    q = randn(gen(seed), len(lens), Hq, D)
    out, sel = call(cache, q, codes, scales, top)
    check(cache, q, codes, scales, top, out, sel)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("top", [1, 2, 3, 8])
def test_edge_lengths(D, top):
    run([0, 1, 15, 16, 17, 31, 32, 33, 48, 49, 64, 100, 127, 128, 129, 500, 1000], top, 8, 2, D, 16, seed=top)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(page, D):
    run([40 * page - 1, 7 * page, 12 * page + 1, 3], 6, 8, 2, D, page, seed=page)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (16, 16), (24, 8), (16, 1), (32, 8), (32, 2)])
def test_head_layouts(Hq, Hkv):
    run([700, 1500], 9, Hq, Hkv, 64, 32, seed=Hq)
    run([700, 1500], 9, Hq, Hkv, 128, 32, seed=Hq)


@pytest.mark.parametrize("top", [17, 33, 64, 100, 257])
def test_many_selected(top):
    run([5000, 4100, 100], top, 8, 2, 64, 16, seed=top)


def test_long_context_and_wide_table():
    run([70000, 1234], 40, 4, 1, 64, 16, seed=1, width=6000)
    run([200003], 64, 2, 1, 64, 16, seed=2)


def test_batch_of_many():
    rng = random.Random(3)
    run([rng.randint(0, 900) for _ in range(70)], 5, 8, 4, 64, 32, seed=3)


def test_ties_go_to_the_lower_page():
    cache = Cache([60 * 16], 1, 64, 16, 4)
    q = randn(gen(4), 1, 4, 64)
    codes = torch.zeros(cache.P, 1, 2, 64, dtype=torch.int8, device="cuda")
    codes[:, :, 1] = 5
    scales = torch.ones(cache.P, 1, device="cuda")
    for level in (None, 7, 30):  # all equal; one page better; one page worse
        if level:
            scales[cache.table[0, level].long()] = 2.0 if level == 7 else 0.5
        out, sel = call(cache, q, codes, scales, 20)
        check(cache, q, codes, scales, 20, out, sel)


def test_scores_that_are_negative_zero_and_huge():
    cache = Cache([40 * 16 + 3], 2, 64, 16, 5)
    g = gen(5)
    q = randn(g, 1, 4, 64)
    codes = torch.randint(-127, -60, (cache.P, 2, 2, 64), generator=g, dtype=torch.int8, device="cuda")
    q[:, :2] = q[:, :2].abs()  # upper bounds below zero for kv head 0
    scales = torch.rand(cache.P, 2, generator=g, device="cuda")
    ids = cache.table[0].long()
    scales[ids[3:6]], scales[ids[9:12]] = torch.finfo(torch.float32).max, 0.0
    codes[ids[9:12]] = 0
    scales[ids[20]] = 1e-42
    out, sel = call(cache, q, codes, scales, 12)
    check(cache, q, codes, scales, 12, out, sel)


@pytest.mark.parametrize("x", [0.0, math.inf, math.nan])
def test_queries_without_a_direction(x):
    cache = Cache([30 * 16], 1, 64, 16, 6)
    codes, scales = summaries(cache)
    q = torch.full((1, 2, 64), x, dtype=torch.bfloat16, device="cuda")
    out, sel = call(cache, q, codes, scales, 5)
    check(cache, q, codes, scales, 5, out, sel, values=x == 0.0)
    if math.isnan(x):
        assert bool(torch.isnan(out).all())


def test_strided_views():
    cache = Cache([900, 333], 2, 64, 32, 7)
    codes, scales = summaries(cache)
    qkv = randn(gen(7), 2, 12, 64)
    hold = torch.zeros(2, 9, 64, dtype=torch.bfloat16, device="cuda")
    out, sel = call(cache, qkv[:, :8], codes, scales, 6, out=hold[:, 1:])
    check(cache, qkv[:, :8], codes, scales, 6, out, sel)
    assert not bool(hold[:, 0].any())


def test_offsets_past_32_bits():
    page, Hkv, D = 64, 8, 64
    pages = (1 << 31) // (Hkv * page * D) + 200
    cache = Cache([3000, 70], Hkv, D, page, 8, pages=pages, base=pages - 100)
    codes, scales = summaries(cache)
    q = randn(gen(8), 2, 16, D)
    out, sel = call(cache, q, codes, scales, 9)
    check(cache, q, codes, scales, 9, out, sel)


def test_bitwise_the_same_again_and_in_another_batch():
    """A sequence's selection and output do not depend on what else is in the batch."""
    cache = Cache([2000, 2000, 17], 2, 64, 16, 9)
    codes, scales = summaries(cache)
    q = randn(gen(9), 3, 8, 64)
    a, sa = call(cache, q, codes, scales, 10)
    b, sb = call(cache, q, codes, scales, 10)
    assert torch.equal(a, b) and torch.equal(sa, sb)
    cache.table, cache.lens = cache.table.flip(0).contiguous(), cache.lens.flip(0).contiguous()
    c, sc = call(cache, q.flip(0).contiguous(), codes, scales, 10)
    assert torch.equal(sc.flip(0), sa) and torch.equal(c.flip(0), a)


def test_all_pages_is_dense_attention():
    cache = Cache([777], 2, 64, 32, 10)
    codes, scales = summaries(cache)
    q = randn(gen(10), 1, 8, 64)
    out, sel = call(cache, q, codes, scales, 25)
    assert sel[0, 0].tolist() == list(range(25))
    ref, tol = attend(q.view(2, 4, 64), cache.K[0], cache.V[0], 0.125)
    assert bool(((out.view(2, 4, 64).double() - ref).abs() <= tol).all())


def test_operator_reference_agrees():
    cache = Cache([300, 40, 0], 2, 64, 16, 11)
    codes, scales = summaries(cache)
    q = randn(gen(11), 3, 8, 64)
    op = PageSelectAttention(batch=3, num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=cache.P, max_pages=cache.M, top_pages=4)
    out, sel = op.reference(*(t.cpu() for t in (q, cache.k, cache.v, codes, scales, cache.table, cache.lens)))
    check(cache, q, codes, scales, 4, out.cuda(), sel.cuda())


@pytest.mark.parametrize("D,pages", [(64, 23500), (128, 26200)])
def test_more_pages_than_keys_fit(D, pages):
    """Sequences whose scores do not fit in shared memory; the second one is short."""
    run([pages * 16 - 11, 100, 0], 40, 8, 2, D, 16, seed=D, width=pages + 3)


@pytest.mark.parametrize("D,width", [(64, None), (128, None), (64, 23500), (128, 26200)])
def test_more_units_than_ctas(D, width):
    """300 (sequence, kv head) units of all lengths: pieces that hold parts of several."""
    rng = random.Random(D)
    lens = [rng.choice([0, 1, 63, 64, 65, 700, 2048, 3000]) for _ in range(150)]
    run(lens, 20, 8, 2, D, 64, seed=D + 1, width=width)
