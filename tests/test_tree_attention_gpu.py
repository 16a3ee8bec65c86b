"""TreeAttention against the formula in float64, row by row, with the derived tolerance of
paged_helpers.attend; every place of the pool that no sequence owns is NaN."""

import math
import random

import pytest
import torch

from paged_helpers import Cache, gen, randn, tree_reference

pytestmark = pytest.mark.gpu

from iron_b200.operators import TreeAttention


def operator(cache, B, N, Hq, scale=None):
    return TreeAttention(batch=B, num_nodes=N, num_heads=Hq, num_kv_heads=cache.Hkv, head_dim=cache.D, page_size=cache.page,
                         num_pages=cache.P, max_pages=cache.M, scale=scale)


def close(out, ref, tol):
    err = (out.double() - ref).abs()
    assert bool(torch.isfinite(out).all())
    assert bool((err <= tol).all()), f"off by {float((err / tol.clamp(min=1e-30)).max()):.2f} times the bound"


def drafted(rng, kind, N):
    if kind == "chain":
        return list(range(-1, N - 1))
    if kind == "star":
        return [-1] * N
    row = [-1] + [rng.randint(-1, i - 1) for i in range(1, N)]
    if kind == "ragged":  # unused places, some of them inside the tree
        for i in rng.sample(range(N), N // 3):
            row[i] = rng.choice([-2, -7, i, i + 1, 1 << 30, -(1 << 31)])
    return row


def run(lens, N, Hq, Hkv, D, page, kind="random", seed=0, scale=None, width=None):
    rng, g = random.Random(seed), gen(seed)
    cache = Cache(lens, Hkv, D, page, seed, width=width)
    B = len(lens)
    qkv = randn(g, B, N, Hq + 2 * Hkv, D)
    q, kn, vn = qkv.split([Hq, Hkv, Hkv], 2)
    parents = [drafted(rng, kind, N) for _ in range(B)]
    out = torch.full((B, N, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda")
    call = operator(cache, B, N, Hq, scale).get_callable()
    call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    ref, tol = tree_reference(cache, q, kn, vn, parents, scale or 1 / math.sqrt(D))
    close(out, ref, tol)
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 255, 257, 511]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [1, 5, 40])
def test_edge_lengths(D, N):
    run(EDGES, N, 8, 2, D, 64, seed=N)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(page, D):
    run([1, 300, page, 3 * page + 1, 777], 9, 8, 2, D, page, seed=page)
    run([1, 300, page, 3 * page + 1, 777], 33, 16, 2, D, page, seed=page + 1)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128])
def test_node_counts(N):
    run([130, 0, 700], N, 8, 2, 64, 64, seed=N)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (16, 16), (24, 8), (16, 1), (32, 8), (32, 2), (10, 2)])
@pytest.mark.parametrize("N,D", [(3, 64), (21, 128)])
def test_head_layouts(Hq, Hkv, N, D):
    run([200, 65, 1], N, Hq, Hkv, D, 32, seed=Hq + N)


@pytest.mark.parametrize("kind", ["chain", "star", "ragged"])
@pytest.mark.parametrize("N", [6, 50, 128])
def test_tree_shapes(kind, N):
    run([0, 90, 400], N, 8, 2, 64, 64, kind=kind, seed=N)


def test_no_node_is_used():
    cache = Cache([0, 100], 2, 64, 64, 1)
    g = gen(1)
    q, kn = randn(g, 2, 5, 8, 64), randn(g, 2, 5, 2, 64)
    out = torch.full_like(q, math.nan)
    parents = torch.tensor([[-2] * 5, [-2, 0, 1, 0, 4]], dtype=torch.int32, device="cuda")
    operator(cache, 2, 5, 8).get_callable()(q, kn, kn, cache.k, cache.v, cache.table, cache.lens, parents, out)
    assert not bool(out.any())


def test_wide_table_and_ragged_batch():
    run([20000, 1, 300, 5000, 0, 64], 12, 8, 2, 64, 64, seed=3, width=4000)
    run([9000, 1, 300], 60, 8, 1, 128, 64, seed=4, width=2000)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [3, 20, 64])
def test_many_tiles_per_piece(N, D):
    """More tiles than the GPU has CTAs: pieces of many tiles, and of several sequences."""
    run([4096, 2999, 2049, 100, 3100, 0, 4000, 640], N, 32, 8, D, 64, seed=N)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [5, 8])
def test_few_rows_and_tables_for_long_sequences(N, D):
    """17 to 32 rows per kv head where full tables would be a lot of work."""
    lens = [0, 1, 700, 2048, 64, 5000, 130, 63, 1025, 16, 400, 129, 2999, 15, 65, 300]
    for kind in ("random", "ragged"):
        run(lens, N, 32, 8, D, 64, kind=kind, seed=N, width=300)


@pytest.mark.parametrize("D", [64, 128])
def test_few_units_in_many_pieces(D):
    run([40001], 2, 1, 1, D, 64, seed=1)
    run([20003, 300], 4, 16, 4, D, 64, seed=2)
    run([30011], 8, 8, 2, D, 64, kind="ragged", seed=3)


@pytest.mark.parametrize("Hq,width", [(8, 16), (32, 16), (32, 1000), (64, 16), (64, 1000)])
@pytest.mark.parametrize("D", [64, 128])
def test_infinite_values_reach_the_rows_that_see_them(Hq, width, D):
    cache = Cache([70, 0, 900, 130], 8, D, 64, 5, width=width)
    g = gen(5)
    q, kn, vn = randn(g, 4, 8, Hq, D), randn(g, 4, 8, 8, D), randn(g, 4, 8, 8, D)
    parents = [[-1, 0, 1, 0, 3, -1, 5, 2]] * 4
    vn[:, 3, :, 7] = math.inf
    vn[:, 6, :, 9] = -math.inf
    out = torch.full_like(q, math.nan)
    operator(cache, 4, 8, Hq).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens,
                                             torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    for n in range(8):
        x = out[:, n].double()
        assert bool((x[..., 7] == math.inf).all()) == (n in (3, 4)) and bool((x[..., 9] == -math.inf).all()) == (n == 6)
        x[..., 7] = x[..., 9] = 0
        assert bool(torch.isfinite(x).all())


# The form for many rows is taken up to 128 rows where tables are wide: the cases above again.
WIDE = 3000


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [9, 20, 32])
def test_edge_lengths_with_wide_tables(D, N):
    run(EDGES, N, 8, 2, D, 64, seed=N, width=WIDE)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes_with_wide_tables(page, D):
    run([1, 300, page, 3 * page + 1, 777], 11, 8, 2, D, page, seed=page, width=4 * WIDE)


@pytest.mark.parametrize("N", [9, 15, 16, 17, 31, 32])
def test_node_counts_with_wide_tables(N):
    run([130, 0, 700], N, 8, 2, 64, 64, seed=N, width=WIDE)


@pytest.mark.parametrize("Hq,Hkv", [(3, 1), (24, 8), (16, 1), (32, 8), (10, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts_with_wide_tables(Hq, Hkv, D):
    run([200, 65, 1], -(-33 * Hkv // Hq), Hq, Hkv, D, 32, seed=Hq, width=4 * WIDE)


@pytest.mark.parametrize("kind", ["chain", "star", "ragged"])
@pytest.mark.parametrize("N,Hq", [(12, 8), (50, 4), (128, 2)])
def test_tree_shapes_with_wide_tables(kind, N, Hq):
    run([0, 90, 400], N, Hq, 2, 64, 64, kind=kind, seed=N, width=WIDE)


@pytest.mark.parametrize("width", [16, 3000])
@pytest.mark.parametrize("D", [64, 128])
def test_broadcast_rows_and_other_scales(D, width):
    """Keys of one batch for all sequences (stride 0), and a scale below zero: many rows
    without the tensor cores' form."""
    cache = Cache([70, 0, 900, 130], 2, D, 64, 5, width=width)
    rng, g = random.Random(2), gen(5)
    N, Hq, scale = 40, 8, -0.07
    q = randn(g, 4, N, Hq, D)
    kn, vn = (randn(g, 1, N, 2, D).expand(4, N, 2, D) for _ in range(2))
    parents = [drafted(rng, "ragged", N) for _ in range(4)]
    table = torch.tensor(parents, dtype=torch.int32, device="cuda")
    for k, v, x in ((kn, vn, None), (kn.contiguous(), vn.contiguous(), scale)):
        out = torch.full_like(q, math.nan)
        operator(cache, 4, N, Hq, x).get_callable()(q, k, v, cache.k, cache.v, cache.table, cache.lens, table, out)
        close(out, *tree_reference(cache, q, k, v, parents, x or 1 / math.sqrt(D)))


def test_batch_of_many():
    rng = random.Random(2)
    run([rng.randint(0, 200) for _ in range(300)], 2, 4, 1, 64, 32, seed=2)


@pytest.mark.parametrize("scale", [4.0, 0.001])
@pytest.mark.parametrize("N", [3, 40])
def test_scale(scale, N):
    run([500, 77], N, 8, 2, 64, 64, seed=5, scale=scale)


@pytest.mark.parametrize("N", [4, 40])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_masked_values_have_no_effect(N, bad):
    """Values that are not finite in nodes off a row's path reach no other row."""
    cache = Cache([100, 0], 2, 64, 64, 1)
    g = gen(N)
    q, kn, vn = randn(g, 2, N, 8, 64), randn(g, 2, N, 2, 64), randn(g, 2, N, 2, 64)
    parents = [[-1] * N, [-1] * N]
    kn[0, 1], vn[1, 2], vn[0, 3, 1, 5] = bad, bad, bad
    kn[:, 0], parents[1][0] = bad, -2  # an unused node's too
    call = operator(cache, 2, N, 8).get_callable()
    out = torch.empty_like(q)
    call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    ref, tol = tree_reference(cache, q, kn, vn, parents, 0.125)
    fine = torch.isfinite(ref)
    assert bool(((out.double() - ref).abs() <= tol)[fine].all())
    # rows that see them are not finite, as the formula's are not
    assert torch.equal(torch.isfinite(out[1]), torch.isfinite(ref[1]))
    assert torch.equal(torch.isfinite(out[0, 3]), torch.isfinite(ref[0, 3]))


@pytest.mark.parametrize("N", [3, 40])
def test_values_at_the_ends_of_the_range(N):
    """A cached token whose logit is far below or above the others."""
    cache = Cache([300], 2, 64, 64, 6)
    g = gen(6)
    q, kn, vn = randn(g, 1, N, 8, 64), randn(g, 1, N, 2, 64), randn(g, 1, N, 2, 64)
    for at, x in ((5, 1e4), (70, -1e4), (299, 3e38)):
        p = int(cache.table[0, at // 64])
        row = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
        row[:, 0] = x
        cache.k[p, :, at % 64] = row
        cache.K[0][:, at] = row
    q[..., 0] = 1.0
    q[0, 0, :, 0] = 0.0
    out = torch.empty_like(q)
    parents = [drafted(random.Random(1), "chain", N)]
    operator(cache, 1, N, 8).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens,
                                            torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    ref, _ = tree_reference(cache, q, kn, vn, parents, 0.125)
    err = (out.double() - ref).abs()
    assert bool((err <= 2.0**-8 * ref.abs().clamp(min=1.0) * 2).all())


@pytest.mark.parametrize("N", [4, 48])
def test_offsets_past_32_bits(N):
    """Pages whose first element lies past 2^31 in the pool."""
    page, Hkv, D = 64, 8, 64
    pages = (1 << 31) // (Hkv * page * D) + 200
    cache = Cache([500, 70], Hkv, D, page, 7, pages=pages, base=pages - 100)
    g = gen(7)
    q, kn, vn = randn(g, 2, N, 8, D), randn(g, 2, N, Hkv, D), randn(g, 2, N, Hkv, D)
    parents = [drafted(random.Random(1), "random", N) for _ in range(2)]
    out = torch.empty_like(q)
    operator(cache, 2, N, 8).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens,
                                            torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    close(out, *tree_reference(cache, q, kn, vn, parents, 0.125))


@pytest.mark.parametrize("N,D", [(6, 64), (64, 64), (64, 128)])
def test_bitwise_the_same_again_and_on_another_stream(N, D):
    cache = Cache([3000, 10, 800], 2, D, 64, 8)
    g = gen(8)
    q, kn, vn = randn(g, 3, N, 8, D), randn(g, 3, N, 2, D), randn(g, 3, N, 2, D)
    parents = torch.tensor([drafted(random.Random(b), "random", N) for b in range(3)], dtype=torch.int32, device="cuda")
    op = operator(cache, 3, N, 8)
    call = op.get_callable()
    a, b, c = (torch.empty_like(q) for _ in range(3))
    call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, parents, a)
    call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, parents, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, parents, c)
    torch.cuda.synchronize()
    assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and torch.equal(a.view(torch.int16), c.view(torch.int16))


def test_strided_output_and_new_rows():
    cache = Cache([150, 20], 2, 64, 64, 9)
    g = gen(9)
    N = 7
    big = randn(g, N, 2, 8, 64)  # node-major
    q = big.transpose(0, 1)
    kv = randn(g, 2, N, 2, 2, 64)  # k and v of a node side by side
    kn, vn = kv[:, :, 0], kv[:, :, 1]
    hold = torch.zeros(2, N, 10, 64, dtype=torch.bfloat16, device="cuda")
    out = hold[:, :, 1:9]
    parents = [drafted(random.Random(b), "random", N) for b in range(2)]
    operator(cache, 2, N, 8).get_callable()(q, kn, vn, cache.k, cache.v, cache.table, cache.lens,
                                            torch.tensor(parents, dtype=torch.int32, device="cuda"), out)
    close(out, *tree_reference(cache, q, kn, vn, parents, 0.125))
    assert not bool(hold[:, :, 0].any()) and not bool(hold[:, :, 9].any())


def test_table_entries_outside_the_pool_are_not_followed():
    cache = Cache([200], 2, 64, 64, 10)
    g = gen(10)
    q, kn = randn(g, 1, 3, 8, 64), randn(g, 1, 3, 2, 64)
    parents = torch.tensor([[-1, 0, 1]], dtype=torch.int32, device="cuda")
    table = cache.table.clone()
    table[0, 1], table[0, 2] = -1, cache.P
    out = torch.empty_like(q)
    operator(cache, 1, 3, 8).get_callable()(q, kn, kn, cache.k, cache.v, table, cache.lens, parents, out)
    keep = list(range(64)) + list(range(192, 200))
    cache.K[0], cache.V[0] = cache.K[0][:, keep], cache.V[0][:, keep]
    close(out, *tree_reference(cache, q, kn, kn, parents.tolist(), 0.125))


def test_operator_reference_agrees():
    cache = Cache([70, 5], 2, 64, 16, 11)
    g = gen(11)
    q, kn, vn = randn(g, 2, 4, 8, 64), randn(g, 2, 4, 2, 64), randn(g, 2, 4, 2, 64)
    parents = torch.tensor([[-1, 0, 0, -2], [-1, -1, 1, 2]], dtype=torch.int32)
    op = operator(cache, 2, 4, 8)
    got = op.reference(*(t.cpu() for t in (q, kn, vn, cache.k, cache.v, cache.table, cache.lens)), parents)
    close(got.cuda(), *tree_reference(cache, q, kn, vn, parents.tolist(), 0.125))
