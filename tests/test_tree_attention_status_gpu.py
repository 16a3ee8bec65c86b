"""A bounded wait of the tcgen05 tree attention that runs out, without faulting the GPU.

With a limit of 0 the loads give up as soon as a slot is not free, so the other roles' data
never comes: each of them ends, the status word is set, and the next call is right again."""

import time

import pytest
import torch

from paged_helpers import Cache, gen, randn, tree_reference
from test_tree_attention_gpu import close, drafted, operator

pytestmark = pytest.mark.gpu

import random

from iron_b200 import _lib
from iron_b200.applications.llama_3_2_1b.decode import LlamaDecodeEngine, LlamaShape
from iron_b200.applications.llama_3_2_1b.paged import PagedDecoder
from iron_b200.operators import TreeAttention


@pytest.fixture
def no_waiting():
    lib = _lib.load()
    lib.iron_tree_attn_status(1)
    yield lambda: lib.iron_tree_attn_set_wait_us(0)
    lib.iron_tree_attn_set_wait_us(2000000)
    lib.iron_tree_attn_status(1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [20, 64])
def test_a_wait_that_runs_out_is_reported(D, N, no_waiting):
    cache = Cache([20000, 0, 700], 8, D, 64, 3, width=400)
    g = gen(3)
    q, kn, vn = randn(g, 3, N, 32, D), randn(g, 3, N, 8, D), randn(g, 3, N, 8, D)
    parents = [drafted(random.Random(b), "random", N) for b in range(3)]
    table = torch.tensor(parents, dtype=torch.int32, device="cuda")
    call = operator(cache, 3, N, 32).get_callable()
    outs = [torch.empty_like(q) for _ in range(2)]
    args = (q, kn, vn, cache.k, cache.v, cache.table, cache.lens, table)
    call(*args, outs[0])
    TreeAttention.check()
    close(outs[0], *tree_reference(cache, q, kn, vn, parents, D**-0.5))
    no_waiting()
    side = torch.cuda.Stream()  # the status waits for the other streams too
    side.wait_stream(torch.cuda.current_stream())
    start = time.perf_counter()
    with torch.cuda.stream(side):
        call(*args, torch.empty_like(q))
    with pytest.raises(RuntimeError, match="timed out"):
        TreeAttention.check()
    assert time.perf_counter() - start < 1.0  # the other roles do not wait for their own limits
    TreeAttention.check()  # reported once
    _lib.load().iron_tree_attn_set_wait_us(2000000)
    call(*args, outs[1])
    TreeAttention.check()
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))


def test_the_decoder_raises_instead_of_going_on(no_waiting):
    # long enough that a piece of the attention has more tiles than the loads have slots
    engine = LlamaDecodeEngine(LlamaShape(n_layers=1, vocab_size=1024), batch=1, max_seq=16384, seed=3, fuse_norm="none")
    d = PagedDecoder(engine, slots=1, nodes=33, num_pages=140, page_size=128)
    prompt = torch.randint(0, 1024, (16000,), generator=torch.Generator().manual_seed(1)).tolist()
    assert len(d.generate([prompt], 2)[0]) == 2
    d.check()
    no_waiting()
    with pytest.raises(RuntimeError, match="timed out"):
        d.generate([prompt], 2)
