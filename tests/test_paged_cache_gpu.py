"""PageAppend, PageFork, PageCompact and PagedKVCache against host integers and moved rows:
everything they write is whole numbers or copies, so all comparisons are exact."""

import math
import random

import pytest
import torch

from paged_helpers import HostCache, gen, randn, summary

pytestmark = pytest.mark.gpu

from iron_b200 import _lib
from iron_b200.operators import PageAppend, PageCompact, PagedKVCache, PageFork


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bits(t):
    return t.view(torch.int16)


class Both:
    """Device buffers and the host's copy of what they must hold."""

    def __init__(self, slots, pages, width, page, layers=2, heads=3, dim=64, seed=0, summaries=False):
        self.host = HostCache(slots, pages, width, page)
        self.sizes = dict(slots=slots, num_layers=layers, num_kv_heads=heads, head_dim=dim, page_size=page, num_pages=pages, max_pages=width)
        self.g = gen(seed)
        self.k, self.v = (randn(self.g, layers, pages, heads, page, dim) for _ in range(2))
        self.K, self.V = self.k.clone(), self.v.clone()
        self.summaries = summaries
        self.codes = torch.full((layers, pages, heads, 2, dim), 77, dtype=torch.int8, device="cuda")
        self.scales = torch.full((layers, pages, heads), 0.5, device="cuda")
        self.C, self.S = self.codes.clone(), self.scales.clone()
        self.push()

    def push(self):
        h = self.host
        self.table, self.lens, self.refs = ints(h.table), ints(h.lens), ints(h.refs)

    def check(self, table, lens, refs):
        assert table.tolist() == self.host.table
        if lens is not None:
            assert lens.tolist() == self.host.lens
        assert refs.tolist() == self.host.refs
        assert torch.equal(bits(self.k), bits(self.K)) and torch.equal(bits(self.v), bits(self.V))
        assert torch.equal(self.codes, self.C) and torch.equal(self.scales, self.S)

    def append(self, index, N, kn=None, alias=False):
        z = self.sizes
        shape = (z["num_layers"], z["slots"], N, z["num_kv_heads"], z["head_dim"])
        kn, vn = randn(self.g, *shape) if kn is None else kn, randn(self.g, *shape)
        takes = [next((j for j, x in enumerate(r) if not 0 <= x < N), N) for r in index]
        refused, wrote = self.host.append(takes)
        full = []
        for s, j, p, r in wrote:
            self.K[:, p, :, r], self.V[:, p, :, r] = kn[:, s, index[s][j]], vn[:, s, index[s][j]]
            full += [p] if r == z["page_size"] - 1 else []
        more = ()
        if self.summaries:
            more = (self.codes, self.scales)
            for p in full:
                codes, scale = summary(self.K[:, p])
                self.C[:, p], self.S[:, p] = codes.to("cuda", torch.int8), scale.cuda()
        out = self.lens if alias else torch.full_like(self.lens, -7)
        status = ints([-1])
        call = PageAppend(**z, num_new=N, summaries=self.summaries).get_callable()
        call(kn, vn, ints(index), self.k, self.v, self.table, self.lens, self.refs, out, status, *more)
        assert int(status) == refused
        self.check(self.table, out, self.refs)
        self.push()
        return refused

    def fork(self, source):
        refused, copies = self.host.fork(source)
        for a, b, r in copies:
            self.K[:, b, :, :r], self.V[:, b, :, :r] = self.k[:, a, :, :r], self.v[:, a, :, :r]
        out = [torch.full_like(t, -9) for t in (self.table, self.lens, self.refs)]
        status = ints([-1])
        PageFork(**self.sizes).get_callable()(ints(source), self.table, self.lens, self.refs, self.k, self.v, *out, status)
        assert int(status) == refused
        self.check(*out)
        self.push()
        return refused

    def compact(self, alias=False):
        used, moves = self.host.compact()
        for a, b in moves:
            self.K[:, b], self.V[:, b] = self.K[:, a].clone(), self.V[:, a].clone()
            if self.summaries:
                self.C[:, b], self.S[:, b] = self.C[:, a].clone(), self.S[:, a].clone()
        table, refs = (self.table, self.refs) if alias else (torch.full_like(self.table, -9), torch.full_like(self.refs, -9))
        word = ints([-1])
        more = (self.codes, self.scales) if self.summaries else ()
        PageCompact(**self.sizes, summaries=self.summaries).get_callable()(self.table, self.refs, self.k, self.v, table, refs, word, *more)
        assert int(word) == used
        self.check(table, None, refs)
        self.push()
        return moves


def linear(takes, N):
    return [list(range(t)) + [-1] * (N - t) for t in takes]


@pytest.mark.parametrize("page,dim,heads", [(16, 64, 1), (32, 128, 3), (64, 64, 8), (128, 128, 2), (64, 128, 33)])
def test_append_lengths(page, dim, heads):
    b = Both(5, 40, 9, page, heads=heads, dim=dim, seed=page)
    assert b.append(linear([0, 1, page - 1, page, page + 1], page + 1), page + 1) == 0
    assert b.append(linear([3, page, 1, 0, 2 * page + 1], 2 * page + 1), 2 * page + 1, alias=True) == 0
    assert b.append([[0], [0], [0], [-1], [0]], 1) == 0


def test_append_picks_rows_of_a_tree():
    b = Both(4, 30, 6, 16, seed=1)
    # the list ends at the first entry outside [0, N), whatever follows; an index may repeat
    assert b.append([[6, 2, 0, -1, 3, 1, 1], [5, 5, 5, 5, 5, 5, 5], [7, 1, 2, 3, 4, 5, 6], [0, 3, 6, -2, -1, -1, -1]], 7) == 0
    assert b.host.lens == [3, 7, 0, 3]


def test_append_refuses_whole_slots():
    b = Both(4, 5, 3, 16, seed=2)
    # 6 pages asked for, 5 there: the slots up to the shortage fit, those that need no page too
    assert b.append(linear([20, 16, 40, 0], 40), 40) == 1
    assert b.host.lens == [20, 16, 0, 0]
    # a table row of 3 pages is full after 48 tokens
    assert b.append(linear([29, 0, 1, 0], 40), 40) == 1
    assert b.host.lens == [20, 16, 1, 0]
    # the pages run out before slot 1; slot 0 still has room in its own page
    b.append(linear([0, 1, 0, 0], 1), 1)
    assert b.append(linear([12, 0, 0, 1], 12), 12) == 1


def test_append_never_writes_a_shared_page():
    b = Both(3, 12, 4, 16, seed=3)
    b.append(linear([32, 0, 0], 32), 32)
    b.fork([0, 0, -1])
    # a rolled-back length would write into a page that slot 1 holds too
    b.host.lens[0] = 20
    b.push()
    assert b.append(linear([1, 1, 0], 1), 1) == 1
    assert b.host.lens == [20, 33, 0]


def test_append_keeps_pages_of_a_rolled_back_slot():
    b = Both(2, 12, 4, 16, seed=4)
    b.append(linear([50, 3], 50), 50)
    b.host.lens[0] = 17
    b.push()
    assert b.append(linear([33, 1], 33), 33) == 0
    assert sum(r > 0 for r in b.host.refs) == 5


@pytest.mark.parametrize("page,dim,heads", [(16, 64, 5), (32, 128, 2), (64, 64, 8), (128, 64, 1)])
def test_append_summaries(page, dim, heads):
    b = Both(4, 30, 5, page, heads=heads, dim=dim, seed=page + 1, summaries=True)
    b.append(linear([page, 3, 2 * page + 5, 0], 2 * page + 5), 2 * page + 5)
    b.append(linear([1, page - 3, page, 0], page), page)  # pages filled in two steps
    kn = randn(b.g, 2, 4, page, heads, dim)
    kn[:, 0] = 0.0  # zero keys
    kn[:, 1, 4, 0, 3] = math.inf
    kn[:, 2, 5, heads - 1, 7] = math.nan
    kn[:, 3] = torch.tensor(1e-40).to(torch.bfloat16)  # subnormal keys
    b.append(linear([page] * 4, page), page, kn=kn)
    b.append(linear([page] * 4, page), page)


def test_append_many_slots_and_pages():
    rng = random.Random(5)
    b = Both(300, 9000, 40, 16, layers=1, heads=1, seed=5)
    b.append(linear([rng.randint(0, 500) for _ in range(300)], 500), 500)
    b.fork([rng.choice([s, -1, -1, s]) for s in range(300)])
    b.append(linear([rng.randint(0, 100) for _ in range(300)], 100), 100)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_fork_random(seed, page, dim):
    rng = random.Random(seed)
    b = Both(9, 80, 7, page, dim=dim, seed=seed)
    b.append(linear([rng.choice([0, 1, page, 2 * page, rng.randint(1, 5 * page)]) for _ in range(9)], 5 * page), 5 * page)
    for _ in range(3):
        b.fork([rng.randint(-1, 8) for _ in range(9)])
        b.append(linear([rng.randint(0, 3) for _ in range(9)], 3), 3)


def test_fork_swaps_and_outside_indices():
    b = Both(4, 20, 4, 16, seed=6)
    b.append(linear([5, 16, 33, 0], 33), 33)
    b.fork([1, 2, 0, 3])  # a permutation moves pages, it copies none
    assert sorted(b.host.refs) == [0] * 15 + [1] * 5 and b.host.lens == [16, 33, 5, 0]
    b.fork([4, 1 << 30, -5, 1])  # outside [0, slots): freed
    assert b.host.lens == [0, 0, 0, 33]


def test_fork_runs_out_of_pages():
    b = Both(4, 4, 4, 16, seed=7)
    b.append(linear([17, 0, 0, 0], 17), 17)
    assert b.fork([0, 0, 0, 0]) == 1
    assert b.host.lens == [17, 17, 17, 0]


def test_fork_gives_back_pages_past_the_length():
    b = Both(2, 10, 5, 16, seed=8)
    b.append(linear([60, 1], 60), 60)
    b.host.lens[0] = 16
    b.push()
    b.fork([0, 1])
    assert sum(b.host.refs) == 2


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("page,heads,summaries", [(16, 1, True), (64, 8, False), (128, 3, True)])
def test_compact_random(page, heads, summaries, alias):
    rng = random.Random(page)
    b = Both(8, 60, 8, page, heads=heads, seed=page, summaries=summaries)
    b.append(linear([rng.randint(0, 7 * page) for _ in range(8)], 7 * page), 7 * page)
    b.fork([0, -1, 2, 0, 2, -1, 2, 7])
    b.append(linear([1] * 8, 1), 1)
    b.fork([-1, 1, 2, 3, -1, 5, 6, -1])
    assert b.compact(alias)
    assert b.compact(alias) == []  # already packed


def test_compact_empty_full_and_large():
    b = Both(2, 6, 3, 16, seed=9)
    b.compact()
    b.append(linear([48, 48], 48), 48)
    b.compact()
    rng = random.Random(9)
    c = Both(64, 30000, 300, 16, layers=1, heads=1, seed=9)
    c.host.table = [[-1] * 300 for _ in range(64)]
    for p in rng.sample(range(30000), 12000):
        row = c.host.table[rng.randrange(64)]
        if -1 in row:
            row[row.index(-1)] = p
            c.host.refs[p] = 1
    c.push()
    assert len(c.compact()) > 3000


@pytest.mark.parametrize("seed", range(3))
def test_cache_holds_what_was_appended(seed):
    """Random appends, forks, frees and compactions; every sequence keeps its tokens."""
    rng, g = random.Random(seed), gen(seed)
    S, layers, heads, page, dim = 6, 2, 2, 16, 64
    c = PagedKVCache(slots=S, num_layers=layers, num_kv_heads=heads, head_dim=dim, page_size=page, num_pages=90, max_pages=12, summaries=True)
    held = [torch.zeros(layers, heads, 0, dim, dtype=torch.bfloat16, device="cuda") for _ in range(S)]
    for _ in range(25):
        what = rng.choice(["append", "append", "fork", "free", "compact"])
        if what == "append":
            n = rng.choice([1, 4, 30])
            kn = randn(g, layers, S, n, heads, dim)
            takes = [rng.randint(0, n) if held[s].shape[2] + n <= 12 * page else 0 for s in range(S)]
            c.append(kn, kn, ints(linear(takes, n)))
            held = [torch.cat([h, kn[:, s, : takes[s]].transpose(1, 2)], 2) for s, h in enumerate(held)]
        elif what == "fork":
            source = [rng.choice([s, rng.randint(0, S - 1)]) for s in range(S)]
            c.fork(ints(source))
            held = [held[r] for r in source]
        elif what == "free":
            s = rng.randrange(S)
            c.free([s])
            held[s] = held[s][:, :, :0]
        else:
            used = int(c.compact())
            assert used == int((c.refs > 0).sum()) and bool((c.refs[:used] > 0).all())
        c.check()
        assert c.lens.tolist() == [h.shape[2] for h in held]
        counts = torch.zeros_like(c.refs)
        counts.scatter_add_(0, c.page_table[c.page_table >= 0].long(), torch.ones_like(c.page_table[c.page_table >= 0]))
        assert torch.equal(counts, c.refs)
        for s, h in enumerate(held):
            n = h.shape[2]
            ids = c.page_table[s, : -(-n // page)].long()
            for pool in (c.k, c.v):
                assert torch.equal(pool[:, ids].transpose(1, 2).reshape(layers, heads, -1, dim)[:, :, :n], h)


def test_cache_reports_refusals():
    c = PagedKVCache(slots=2, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16, num_pages=1, max_pages=2)
    kn = torch.zeros(1, 2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    c.append(kn, kn, ints(linear([4, 4], 4)))
    with pytest.raises(RuntimeError, match="1 slot"):
        c.check()
    c.check()
    assert c.lens.tolist() == [4, 0]


def test_operators_replay_in_a_graph_on_another_stream():
    b = Both(3, 20, 4, 16, seed=11)
    b.append(linear([17, 3, 0], 17), 17)
    op = PageAppend(**b.sizes, num_new=2)
    kn, vn = randn(b.g, 2, 3, 2, 3, 64), randn(b.g, 2, 3, 2, 3, 64)
    index, status = ints(linear([2, 1, 2], 2)), ints([0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        op.prepare()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.get_callable()(kn, vn, index, b.k, b.v, b.table, b.lens, b.refs, b.lens, status)
    torch.cuda.synchronize()
    assert b.lens.tolist() == [17, 3, 0]  # captured, not run
    for _ in range(3):
        graph.replay()
        _, wrote = b.host.append([2, 1, 2])
        for s, j, p, r in wrote:
            b.K[:, p, :, r], b.V[:, p, :, r] = kn[:, s, j], vn[:, s, j]
    torch.cuda.synchronize()
    b.check(b.table, b.lens, b.refs)


def test_fork_refuses_overlapping_state():
    b = Both(2, 4, 2, 16)
    out = [torch.empty_like(t) for t in (b.table, b.lens, b.refs)]
    call = PageFork(**b.sizes).get_callable()
    with pytest.raises(RuntimeError, match="invalid argument"):
        call(ints([0, 1]), b.table, b.lens, b.refs, b.k, b.v, b.table, out[1], out[2], ints([0]))
    with pytest.raises(RuntimeError, match="invalid argument"):
        call(ints([0, 1]), b.table, b.lens, b.refs, b.k, b.v, out[0], out[1], b.refs, ints([0]))
