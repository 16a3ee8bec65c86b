"""TreeAttention with 33 to 128 rows per kv head, where the two streams of the tcgen05 form
take turns at the tiles: batches whose pieces start with one tile, hold several units or
runs of empty sequences. Each is compared with float64 and then called a hundred times: every
call gives the same bits, and no bounded wait runs out."""

import random

import pytest
import torch

from paged_helpers import Cache, gen, randn, tree_reference
from test_tree_attention_gpu import close, drafted, operator

pytestmark = pytest.mark.gpu

from iron_b200 import _lib

BATCHES = {
    "many tiles per piece": [4096, 2999, 2049, 100, 3100, 0, 4000, 640],
    "uniform": [2048] * 16,
    "ragged": [random.Random(1).randint(1, 4096) for _ in range(40)],
    "empty slots": [0] * 8 + [700, 0, 0, 0, 1500, 128] + [0] * 20 + [64, 65, 3000],
    "all empty": [0] * 64,
}


def repeat(lens, N, Hq, Hkv, D, width=64, calls=100):
    rng, g = random.Random(N), gen(N)
    cache = Cache(lens, Hkv, D, 64, N, width=width)
    B = len(lens)
    qkv = randn(g, B, N, Hq + 2 * Hkv, D)
    q, kn, vn = qkv.split([Hq, Hkv, Hkv], 2)
    parents = [drafted(rng, "ragged", N) for _ in range(B)]
    table = torch.tensor(parents, dtype=torch.int32, device="cuda")
    call = operator(cache, B, N, Hq).get_callable()
    _lib.load().iron_tree_attn_status(1)
    first = torch.empty(B, N, Hq, D, dtype=torch.bfloat16, device="cuda")
    call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, table, first)
    close(first, *tree_reference(cache, q, kn, vn, parents, D**-0.5))
    differ = torch.zeros((), dtype=torch.int32, device="cuda")
    for _ in range(calls):
        out = torch.full_like(first, float("nan"))
        call(q, kn, vn, cache.k, cache.v, cache.table, cache.lens, table, out)
        differ += (out.view(torch.int16) != first.view(torch.int16)).any()
    assert int(differ) == 0
    assert _lib.load().iron_tree_attn_status(1) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,Hq", [(11, 24), (20, 32), (32, 32)])
@pytest.mark.parametrize("batch", BATCHES)
def test_every_call_is_the_same(batch, N, Hq, D):
    repeat(BATCHES[batch], N, Hq, 8, D)


@pytest.mark.parametrize("D", [64, 128])
def test_long_sequences_beside_empty_slots(D):
    repeat([16390, 0, 31000, 0, 20001, 25000, 32768], 9, 32, 8, D, width=520)
