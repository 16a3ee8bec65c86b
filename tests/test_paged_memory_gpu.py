"""Appends of many different lengths keep one workspace, not one per length."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from iron_b200.applications.llama_3_2_1b.decode import LlamaDecodeEngine, LlamaShape
from iron_b200.applications.llama_3_2_1b.paged import PagedDecoder
from iron_b200.operators import PagedKVCache


def test_cache_appends_of_many_lengths():
    pages = 1 << 18  # a workspace of 1 MiB
    c = PagedKVCache(slots=2, num_layers=1, num_kv_heads=1, head_dim=64, page_size=16, num_pages=pages, max_pages=100)
    kn = torch.zeros(1, 2, 40, 1, 64, dtype=torch.bfloat16, device="cuda")
    index = torch.arange(40, dtype=torch.int32, device="cuda").repeat(2, 1)

    def append(n):
        c.append(kn[:, :, :n].contiguous(), kn[:, :, :n].contiguous(), index[:, :n].contiguous())

    append(1)
    before = torch.cuda.memory_allocated()
    for n in range(2, 41):
        append(n)
    c.check()
    assert c.lens.tolist() == [820, 820]
    assert torch.cuda.memory_allocated() - before < pages * 4


def test_prompts_of_many_lengths():
    engine = LlamaDecodeEngine(LlamaShape(n_layers=1, vocab_size=1024), batch=1, max_seq=64, seed=3, fuse_norm="none")
    pages = 1 << 14  # a workspace of 64 KiB
    d = PagedDecoder(engine, slots=1, nodes=1, num_pages=pages, page_size=16)
    for n in (40, 19, 40):
        d.prefill([1] * n, 0)
        d.cache.free([0])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for n in [*range(20, 40), 40]:  # (the engine's own buffers are those of the last prompt)
        d.prefill([1] * n, 0)
        d.cache.free([0])
    torch.cuda.synchronize()
    more = torch.cuda.memory_allocated() - before
    assert more < 4 * pages * 4, more
