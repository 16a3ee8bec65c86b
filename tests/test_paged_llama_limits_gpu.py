"""The paged decoder at the ends of its room: sequences past the engine's own cache, outputs
that exactly fill the table, refusals."""

import pytest
import torch

from test_paged_llama_gpu import TOL, agree, plain_logits, prompt

pytestmark = pytest.mark.gpu

from iron_b200.applications.llama_3_2_1b.decode import LlamaDecodeEngine, LlamaShape
from iron_b200.applications.llama_3_2_1b.paged import PagedDecoder

SHAPE = dict(n_layers=2, vocab_size=4096)


@pytest.fixture(scope="module")
def engine():
    return LlamaDecodeEngine(LlamaShape(**SHAPE), batch=1, max_seq=310, seed=3, fuse_norm="none")


@pytest.fixture(scope="module")
def longer():
    """The same weights with room for more tokens."""
    return LlamaDecodeEngine(LlamaShape(**SHAPE), batch=1, max_seq=480, seed=3, fuse_norm="none")


def same_keys(decoder, engine, first, last):
    """The cached keys of tokens first .. last - 1 (of both layers) are those of the plain decode."""
    c = decoder.cache
    ids = c.page_table[0, : -(-last // 16)].long()
    got = c.k[:, ids].transpose(1, 2).flatten(2, 3)[:, :, first:last].float()
    ref = engine.kc[:, 0, :, first:last].float()
    assert float(((got - ref).norm(dim=-1) / ref.norm(dim=-1)).max()) < TOL


def test_drafts_past_the_engines_tokens_are_rotated_by_their_own_angles(engine, longer):
    d = PagedDecoder(engine, slots=1, nodes=8, num_pages=40, page_size=16, max_pages=30)
    text = prompt(307, 1)
    d.prefill(text, 0)
    new = prompt(24, 2)
    ref = plain_logits(longer, text + new, len(text))
    parents = torch.tensor([list(range(-1, 7))], dtype=torch.int32, device="cuda")
    for at in range(0, 24, 8):  # positions 307 to 330
        d.verify(torch.tensor([new[at : at + 8]], dtype=torch.int32, device="cuda"), parents)
        agree(d.logits.float(), ref[at : at + 8])
        d.accept([list(range(8))])
    d.cache.check()
    same_keys(d, longer, len(text), len(text) + len(new) - 1)


def test_selected_decode_past_the_engines_tokens(engine, longer):
    d = PagedDecoder(engine, slots=1, nodes=1, num_pages=40, page_size=16, max_pages=30)
    text, new = prompt(305, 3), prompt(12, 4)
    d.prefill(text, 0)
    rows = []
    for t in new:
        d.decode_selected(torch.tensor([t], dtype=torch.int32, device="cuda"))
        rows.append(d.logits[0].float().clone())
    agree(torch.stack(rows), plain_logits(longer, text + new, len(text)))
    same_keys(d, longer, len(text), len(text) + len(new) - 1)


def drafts_from(monkeypatch, known):
    """generate drafts what is known of the text as a chain (all of it is accepted)."""

    def draft(text, nodes):
        chain = [text[-1]] + known[len(text) : len(text) + nodes - 1]
        pad = nodes - len(chain)
        return chain + [0] * pad, list(range(-1, len(chain) - 1)) + [-2] * pad

    monkeypatch.setattr("iron_b200.applications.llama_3_2_1b.paged.lookup_draft", draft)


@pytest.mark.parametrize("max_new", [2, 9, 20, 22])
def test_output_that_just_fits_does_not_depend_on_lucky_drafts(engine, monkeypatch, max_new):
    """The last pass may accept more than is wanted: those rows need no room."""
    text = prompt(300, 5)
    d = PagedDecoder(engine, slots=1, nodes=8, num_pages=40, page_size=16, max_pages=30)
    out = d.generate([text], 40)[0]
    known = text + out
    small = PagedDecoder(engine, slots=1, nodes=8, num_pages=20, page_size=16, max_pages=20)  # 320 tokens
    drafts_from(monkeypatch, known)
    assert small.generate([text], max_new)[0] == out[:max_new]
    assert small.passes <= -(-max_new // 8) + 1  # the drafts were accepted
    small.cache.check()
    assert not bool(small.cache.refs.any())
    assert small.generate([text], max_new, stop=out[1])[0] == out[: min(max_new, out.index(out[1]) + 1)]


def test_a_refused_slot_ends_generate_at_once(engine, monkeypatch):
    """Pages run out in the middle: the text must not go on over a cache that lacks its rows."""
    text = prompt(40, 6)
    d = PagedDecoder(engine, slots=1, nodes=8, num_pages=3, page_size=16)
    drafts_from(monkeypatch, [])
    with pytest.raises(RuntimeError, match="refused"):
        d.generate([text], 60)
    assert d.passes == 9  # 8 tokens fit the third page
    assert len(d.generate([text], 9)[0]) == 9  # and the decoder is usable


def test_a_refusal_from_before_is_raised_before_generate_starts(engine):
    d = PagedDecoder(engine, slots=1, nodes=8, num_pages=2, page_size=16)
    d.prefill(prompt(30, 7), 0)
    d.verify(*(torch.zeros(1, 8, dtype=torch.int32, device="cuda") - i for i in (0, 1)))
    d.accept([list(range(8))])
    d.passes = -1
    with pytest.raises(RuntimeError, match="refused"):
        d.generate([prompt(10, 8)], 2)
    assert d.passes == -1
    assert len(d.generate([prompt(10, 8)], 2)[0]) == 2


def test_a_refused_selected_step_moves_no_slot(engine):
    d = PagedDecoder(engine, slots=2, nodes=1, num_pages=2, page_size=16)
    texts = [prompt(16, 9), prompt(5, 10)]
    for i, t in enumerate(texts):
        d.prefill(t, i)
    step = torch.tensor([7, 9], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="refused"):
        d.decode_selected(step)  # slot 0 needs a third page
    assert d.cache.lens.tolist() == [16, 5]
    d.cache.free([0])
    d.decode_selected(step)
    assert d.cache.lens.tolist() == [1, 6]
    agree(d.logits[1:].float(), plain_logits(engine, texts[1] + [9], 5))


def test_a_prompt_needs_an_empty_slot(engine):
    """Its keys are rotated for positions 0, 1, ...; behind other tokens they would be wrong."""
    d = PagedDecoder(engine, slots=2, nodes=1, num_pages=8, page_size=16)
    d.prefill(prompt(20, 11), 1)
    with pytest.raises(ValueError, match="slot 1 holds 20 tokens"):
        d.prefill(prompt(5, 12), 1)
    for slot in (-1, 2):
        with pytest.raises(ValueError, match="slot must be"):
            d.prefill(prompt(5, 12), slot)
    assert d.cache.lens.tolist() == [0, 20]
    d.cache.free([1])
    d.prefill(prompt(5, 12), 1)
    assert d.cache.lens.tolist() == [0, 5]


def test_a_wide_table_takes_no_memory_for_angles(engine):
    """A slot holds no more tokens than the pool has, however wide its table row is."""
    d = PagedDecoder(engine, slots=1, nodes=3, num_pages=8, page_size=16, max_pages=100000, top_pages=4)
    assert d._lut.shape[0] == 8 * 16 + 3
    text = prompt(120, 13)
    assert d.generate([text], 9)[0] == PagedDecoder(engine, slots=1, nodes=3, num_pages=8, page_size=16).generate([text], 9)[0]
