"""TreeAttention in CUDA graphs that replay beside other calls of the same operator."""

import random

import pytest
import torch

from paged_helpers import Cache, gen, randn, tree_reference
from test_tree_attention_gpu import close, drafted, operator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,D", [(4, 64), (8, 128), (64, 64)])
def test_graphs_and_eager_calls_side_by_side(N, D):
    """Two graphs captured on the same stream without prepare(), the second replayed first, and
    eager calls on the default stream and the capture stream between replays on others."""
    cache = Cache([3000, 0, 801], 2, D, 64, 5)
    g = gen(5)
    q, kn, vn = randn(g, 3, N, 8, D), randn(g, 3, N, 2, D), randn(g, 3, N, 2, D)
    parents = [drafted(random.Random(b), "random", N) for b in range(3)]
    table = torch.tensor(parents, dtype=torch.int32, device="cuda")
    call = operator(cache, 3, N, 8).get_callable()
    outs = [torch.zeros_like(q) for _ in range(5)]
    run = lambda i: call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, table, outs[i])  # noqa: E731
    graphs, streams = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.cuda.Stream() for _ in range(3)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, stream=streams[2]):
            run(i)
            run(i)
    torch.cuda.synchronize()
    ref, tol = tree_reference(cache, q, kn, vn, parents, D**-0.5)
    graphs[1].replay()
    torch.cuda.synchronize()
    close(outs[1], ref, tol)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(40):
        for i in (1, 0):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            run(2)
        run(3)
    torch.cuda.synchronize()
    run(4)
    for out in outs:
        close(out, ref, tol)
        assert torch.equal(out.view(torch.int16), outs[1].view(torch.int16))


def test_a_graph_is_released_with_its_memory():
    cache = Cache([500], 2, 64, 64, 6)
    g = gen(6)
    q, kn = randn(g, 1, 64, 8, 64), randn(g, 1, 64, 2, 64)
    table = torch.tensor([drafted(random.Random(1), "random", 64)], dtype=torch.int32, device="cuda")
    op = operator(cache, 1, 64, 8)
    call, out = op.get_callable(), torch.empty_like(q)
    call(q, kn, kn, cache.k, cache.v, cache.table, cache.lens, table, out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(q, kn, kn, cache.k, cache.v, cache.table, cache.lens, table, out)
        graph.replay()
        torch.cuda.synchronize()
        del graph
    call(q, kn, kn, cache.k, cache.v, cache.table, cache.lens, table, out)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() <= before
