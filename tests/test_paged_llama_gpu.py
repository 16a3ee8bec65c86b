"""The paged decoder (speculative trees, selected pages) against the engine's plain decode of
the same tokens. Both run the model in bf16 with one rounding per kernel, but other kernels
for other batch sizes, so single values may differ by an ulp (2^-7) that later layers carry
on; over a row of logits such differences are independent, and 8 roundings in each of 2
layers leave them below sqrt(16) 2^-8 = 0.016 of the row's norm, twice that between two
such runs. Predictions are compared where the plain decode's best two logits differ by more
than that share of the best."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from iron_b200.applications.llama_3_2_1b.decode import LlamaDecodeEngine, LlamaShape
from iron_b200.applications.llama_3_2_1b.paged import PagedDecoder, accepted_path, lookup_draft

TOL = 2 * 16**0.5 * 2.0**-8


@pytest.fixture(scope="module")
def engine():
    return LlamaDecodeEngine(LlamaShape(n_layers=2, vocab_size=4096), batch=1, max_seq=320, seed=3, fuse_norm="none")


def prompt(n, seed):
    return torch.randint(0, 4096, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def plain_logits(engine, text, first):
    """Logits of the plain decode after positions first .. len(text) - 1 of text."""
    engine.prefill(text[:first], 0)
    rows = []
    for i in range(first, len(text)):
        engine.set_state([text[i]], [i])
        engine.step()
        rows.append(engine.logits[0].float().clone())
    return torch.stack(rows)


def agree(got, ref):
    off = (got - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert float(off.max()) < TOL, off
    best = ref.topk(2, -1).values
    sure = (best[:, 0] - best[:, 1]) > TOL * best[:, 0].abs()
    assert torch.equal(got.argmax(-1)[sure], ref.argmax(-1)[sure])


def test_a_tree_gives_each_path_its_own_logits(engine):
    d = PagedDecoder(engine, slots=2, nodes=7, num_pages=20, page_size=16)
    texts = [prompt(37, 1), prompt(80, 2)]
    for i, t in enumerate(texts):
        d.prefill(t, i)
    tokens = [[11, 12, 13, 14, 15, 16, 17], [21, 22, 23, 24, 0, 0, 0]]
    parents = [[-1, 0, 0, 1, 1, 3, 2], [-1, 0, 1, 2, -2, -2, -2]]
    d.verify(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (tokens, parents)))
    logits = d.logits.view(2, 7, -1).float().clone()
    for b, leaves in ((0, (5, 4, 6)), (1, (3,))):
        for leaf in leaves:
            path = []
            while leaf >= 0:
                path.append(leaf)
                leaf = parents[b][leaf]
            path.reverse()
            agree(logits[b, path], plain_logits(engine, texts[b] + [tokens[b][i] for i in path], len(texts[b])))


def test_generate_is_the_plain_greedy_decode(engine):
    d = PagedDecoder(engine, slots=3, nodes=8, num_pages=40, page_size=16)
    # the second prompt repeats itself, so that lookups find something
    prompts = [prompt(40, 4), prompt(12, 5) * 4, prompt(5, 6)]
    out = d.generate(prompts, 24)
    for p, o in zip(prompts, out):
        assert len(o) == 24
        ref = plain_logits(engine, p + o[:-1], len(p))  # the prediction after p itself is the prefill's
        best = ref.topk(2, -1).values
        sure = (best[:, 0] - best[:, 1]) > TOL * best[:, 0].abs()
        assert torch.equal(ref.argmax(-1).cpu()[sure.cpu()], torch.tensor(o[1:])[sure.cpu()])
    assert not bool(d.cache.refs.any()) and not bool(d.cache.lens.any())  # everything was freed


def test_a_known_draft_is_accepted_whole(engine):
    d = PagedDecoder(engine, slots=1, nodes=8, num_pages=20, page_size=16)
    p = prompt(30, 7)
    out = d.generate([p], 17)[0]
    passes = d.passes
    d.cache.free([0])
    first = d.prefill(p, 0)
    assert first == out[0]
    # the known continuation as a chain with a wrong sibling at every step
    tokens, parents = [out[0]], [-1]
    for t in out[1:4]:
        parents += [parents.index(-1) if len(tokens) == 1 else len(tokens) - 1] * 2
        tokens += [(t + 1) % 4096, t]
    tokens, parents = tokens + [0], parents + [-2]
    pred = d.verify(*(torch.tensor([x], dtype=torch.int32, device="cuda") for x in (tokens, parents)))[0].tolist()
    path = accepted_path(tokens, parents, pred)
    assert [tokens[i] for i in path] == out[:4] and pred[path[-1]] == out[4]
    d.accept([path])
    assert d.cache.lens.tolist() == [34] and passes <= 17


def test_forks_continue_alike_and_survive_compaction(engine):
    d = PagedDecoder(engine, slots=4, nodes=4, num_pages=24, page_size=16)
    p = prompt(45, 8)
    t = d.prefill(p, 2)
    src = torch.tensor([2, -1, 2, 2], dtype=torch.int32, device="cuda")
    d.cache.fork(src)
    assert d.cache.lens.tolist() == [45, 0, 45, 45]
    tokens = torch.tensor([[t, 5, 6, 7]] * 4, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, 1, 2]] * 4, dtype=torch.int32, device="cuda")
    parents[1] = -2
    d.verify(tokens, parents)
    a = d.logits.view(4, 4, -1).clone()
    assert torch.equal(a[0], a[2]) and torch.equal(a[0], a[3])
    d.accept([[0, 1], [], [0], [0, 1, 2, 3]])
    d.cache.free([0])
    used = int(d.cache.compact())
    assert used == int((d.cache.refs > 0).sum())
    d.cache.check()
    assert d.cache.lens.tolist() == [0, 0, 46, 49]
    d.verify(tokens, torch.tensor([[-2] * 4, [-2] * 4, [-1, 0, 1, 2], [-1, 0, 1, 2]], dtype=torch.int32, device="cuda"))
    got = d.logits.view(4, 4, -1).float()
    for b, text in ((2, p + [t]), (3, p + [t, 5, 6, 7])):
        agree(got[b], plain_logits(engine, text + [t, 5, 6, 7], len(text)))


def test_selected_decode_with_every_page_is_the_plain_decode(engine):
    d = PagedDecoder(engine, slots=2, nodes=1, num_pages=40, page_size=16)
    texts = [prompt(60, 9), prompt(33, 10)]
    new = [prompt(20, 11), prompt(20, 12)]
    for i, t in enumerate(texts):
        d.prefill(t, i)
    rows = []
    for j in range(20):
        d.decode_selected(torch.tensor([n[j] for n in new], dtype=torch.int32, device="cuda"))
        rows.append(d.logits.float().clone())
    assert d.cache.lens.tolist() == [80, 53]
    for b in range(2):
        agree(torch.stack([r[b] for r in rows]), plain_logits(engine, texts[b] + new[b], len(texts[b])))


def test_selected_decode_reads_the_pages_it_names(engine):
    d = PagedDecoder(engine, slots=1, nodes=1, num_pages=40, page_size=16, top_pages=4)
    d.prefill(prompt(200, 13), 0)
    for j in range(3):
        d.decode_selected(torch.tensor([100 + j], dtype=torch.int32, device="cuda"))
        for picked in d.selected[0].tolist():
            assert picked[0] == 0 and picked[-1] == (200 + j) // 16 and len(set(picked)) == 4


def test_lookup_and_refusals(engine):
    assert lookup_draft([1, 2, 3, 1], 4) == ([1, 2, 3, 1], [-1, 0, 1, 2])
    assert lookup_draft([5], 3) == ([5, 0, 0], [-1, -2, -2])
    tokens, parents = lookup_draft([1, 2, 9, 1, 2, 3, 1], 6)  # the latest follow-up first, then a branch of the other
    assert (tokens, parents) == ([1, 2, 3, 1, 9, 1], [-1, 0, 1, 2, 1, 4])
    with pytest.raises(ValueError):
        PagedDecoder(engine, slots=9, nodes=8, num_pages=4)
    d = PagedDecoder(engine, slots=1, nodes=1, num_pages=1, page_size=16)
    with pytest.raises(RuntimeError, match="does not fit"):
        d.prefill(prompt(17, 1), 0)
    with pytest.raises(ValueError):
        d.generate([[1], [2]], 3)
