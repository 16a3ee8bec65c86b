"""Speculative and long-context decode of Llama-3.2-1B over a paged KV cache.

`PagedDecoder` runs the weights of a `LlamaDecodeEngine` (the decode step of
iron/applications/llama_3.2_1b/llama_npu.py:459-584) on a `PagedKVCache`:

- ``prefill`` puts a prompt into a slot's pages;
- ``verify`` runs a drafted tree of tokens per slot through the model in one pass
  (TreeAttention; the drafts' keys and values stay outside the cache), ``accept`` appends
  the longest path the model agrees with (PageAppend);
- ``decode_selected`` decodes one token per slot over the pages that PageSelectAttention
  picks;
- ``cache.fork`` / ``free`` / ``compact`` share, reorder, drop and pack the slots.

``generate`` puts them together: greedy speculative decoding with drafts looked up in the
text so far.

    engine = LlamaDecodeEngine(LlamaShape(), batch=1, max_seq=4096)
    decoder = PagedDecoder(engine, slots=4, nodes=8, num_pages=512)
    texts = decoder.generate([prompt_ids, ...], max_new=64)
"""

from __future__ import annotations

import torch

from ... import _lib
from ...operators import PageAppend, PagedKVCache, PageSelectAttention, TreeAttention
from .decode import LlamaDecodeEngine, rope_table


def lookup_draft(text, nodes: int):
    """(tokens, parents) of a draft: the root, text's last token, and what followed its last
    occurrences in the text -- the latest one as a chain, earlier ones as branches of the
    root while places are left. Unused places have parent -2."""
    tokens, parents = [text[-1]], [-1]
    for at in range(len(text) - 2, -1, -1):
        if len(tokens) == nodes:
            break
        if text[at] != text[-1]:
            continue
        follow, node = text[at + 1 : at + 1 + nodes], 0
        for t in follow:
            child = next((i for i in range(len(tokens)) if parents[i] == node and tokens[i] == t), None)
            if child is None:
                if len(tokens) == nodes:
                    break
                tokens.append(t)
                parents.append(node)
                child = len(tokens) - 1
            node = child
    pad = nodes - len(tokens)
    return tokens + [0] * pad, parents + [-2] * pad


def accepted_path(tokens, parents, predicted):
    """The nodes from the root on whose every token is what the model predicts at its parent."""
    path = [0]
    while True:
        nxt = next((i for i in range(len(tokens)) if parents[i] == path[-1] and tokens[i] == predicted[path[-1]]), None)
        if nxt is None:
            return path
        path.append(nxt)


class PagedDecoder:
    def __init__(self, engine: LlamaDecodeEngine, slots: int, nodes: int, num_pages: int, page_size: int = 64,
                 max_pages: int | None = None, top_pages: int | None = None):
        """nodes: drafted tokens per slot and pass, the root included (slots * nodes <= 64, the
        int4 GEMV's vectors); max_pages: pages of a slot (those of the engine's max_seq tokens
        unless given; a slot may grow past max_seq, only a prompt may not); top_pages: pages that
        decode_selected reads per kv head."""
        if not 1 <= slots * nodes <= 64:
            raise ValueError(f"slots * nodes must be 1 to 64, got {slots} * {nodes}")
        self.engine, self.s, self.slots, self.nodes = engine, engine.s, slots, nodes
        s = self.s
        max_pages = max_pages or -(-engine.L // page_size)
        self.cache = PagedKVCache(slots=slots, num_layers=s.n_layers, num_kv_heads=s.n_kv_groups, head_dim=s.head_dim,
                                  page_size=page_size, num_pages=num_pages, max_pages=max_pages, summaries=True)
        sizes = dict(num_heads=s.n_heads, num_kv_heads=s.n_kv_groups, head_dim=s.head_dim, page_size=page_size,
                     num_pages=num_pages, max_pages=max_pages)
        self._tree = TreeAttention(batch=slots, num_nodes=nodes, **sizes).get_callable()
        top = min(top_pages or max_pages, 4096)
        self._select = PageSelectAttention(batch=slots, top_pages=top, **sizes).get_callable()
        sizes.pop("num_heads")
        self._layer_append = PageAppend(slots=slots, num_layers=1, num_new=1, summaries=True, **sizes).get_callable()
        # prompts: one operator per length, on shared workspaces
        self._row_append, self._row_sizes = {}, dict(slots=1, num_layers=s.n_layers, summaries=True, **sizes)
        self._first_row = PageAppend(**self._row_sizes)
        dev, bf = engine.dev, dict(dtype=torch.bfloat16, device=engine.dev)
        # angles of every position that a slot and the drafts behind it can have (a table may be
        # wider than the pool)
        self._lut = rope_table(s.head_dim, min(max_pages, num_pages) * page_size + nodes, s.rope_base, dev)
        R = slots * nodes
        self._x, self._xn, self._h = (torch.zeros(R, s.emb_dim, **bf) for _ in range(3))
        self._qkv, self._rot = (torch.zeros(R, s.n_heads + 2 * s.n_kv_groups, s.head_dim, **bf) for _ in range(2))
        self._attn, self._act = torch.zeros(R, s.n_heads, s.head_dim, **bf), torch.zeros(R, s.hidden_dim, **bf)
        self.logits = torch.zeros(R, s.vocab_size, **bf)
        self._k, self._v = (torch.zeros(s.n_layers, slots, nodes, s.n_kv_groups, s.head_dim, **bf) for _ in range(2))
        self._ints = dict(dtype=torch.int32, device=dev)
        self._pred = torch.zeros(R, **self._ints)
        self._scratch = torch.zeros(slots, **self._ints)
        self._status = torch.zeros(1, **self._ints)
        # the pages that the last layer of decode_selected read, [slots, kv heads, top_pages]
        self.selected = torch.full((slots, s.n_kv_groups, top), -1, **self._ints)

    # -- the model around the attention ----------------------------------------------------
    def _forward(self, tokens, positions, attend):
        """Logits and greedy predictions of R tokens at their positions; attend(layer, q, k, v,
        out) is the attention of one layer."""
        e, s, st = self.engine, self.s, _lib.current_stream()
        call, p = _lib.call, (lambda t: t.data_ptr())
        R, E, D, Hq, G = tokens.numel(), s.emb_dim, s.head_dim, s.n_heads, s.n_kv_groups
        x, xn, h, qkv, rot, attn, act = (t[:R] for t in (self._x, self._xn, self._h, self._qkv, self._rot, self._attn, self._act))
        call("iron_embed", p(tokens), p(e.embed_table), p(x), R, E, s.vocab_size, 0, st)
        for li, lay in enumerate(e.layers):
            call("iron_rmsnorm", p(x), None, None, p(lay["n1"]), p(xn), R, E, s.eps, 0, st)
            call("iron_gemv_int4g32", p(lay["qkv"].packed), p(xn), p(qkv), s.qkv_dim, E, R, None, 0, st)
            # every head of a token is rotated by the token's angle; v is taken from qkv
            call("iron_rope", p(qkv), None, p(self._lut), p(rot), R * (Hq + 2 * G), D, R, p(positions), 0, 0, st)
            attend(li, rot[:, :Hq], rot[:, Hq : Hq + G], qkv[:, Hq + G :], attn)
            call("iron_gemv_int4g32", p(lay["o"].packed), p(attn), p(h), E, Hq * D, R, p(x), 0, st)
            call("iron_rmsnorm", p(h), None, None, p(lay["n2"]), p(xn), R, E, s.eps, 0, st)
            call("iron_gemv_int4g32", p(lay["gu"].packed), p(xn), p(act), 2 * s.hidden_dim, E, R, None,
                 _lib.IRON_FLAG_SWIGLU, st)
            call("iron_gemv_int4g32", p(lay["d"].packed), p(act), p(x), E, s.hidden_dim, R, p(h), 0, st)
        call("iron_rmsnorm", p(x), None, None, p(e.nf), p(xn), R, E, s.eps, 0, st)
        call("iron_gemv_int4g32", p(e.lm.packed), p(xn), p(self.logits), s.vocab_size, E, R, None, 0, st)
        call("iron_argmax", p(self.logits), p(self._pred), R, s.vocab_size, None, 0, st)
        return self._pred[:R]

    def _in_table(self, positions):
        """Positions that the operators' own lengths never pass, whatever someone wrote there."""
        return positions.clamp(0, self._lut.shape[0] - 1)

    # -- cache ---------------------------------------------------------------------------------
    def prefill(self, tokens, slot: int):
        """Runs a prompt through the engine and puts its keys and values into the slot's pages
        (ValueError if the slot is not empty). Returns the model's next token."""
        e, c, n = self.engine, self.cache, len(tokens)
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot must be 0 to {self.slots - 1}, got {slot}")
        if int(c.lens[slot]):
            raise ValueError(f"slot {slot} holds {int(c.lens[slot])} tokens: free it first")
        e.prefill(tokens, 0)
        if n not in self._row_append:
            op = PageAppend(num_new=n, **self._row_sizes)
            self._row_append[n] = op.share_workspaces(self._first_row).get_callable()
        k, v = (x[:, 0, :, :n].transpose(1, 2).contiguous() for x in (e.kc, e.vc))
        row = slice(slot, slot + 1)
        index = torch.arange(n, **self._ints)
        self._row_append[n](k, v, index, c.k, c.v, c.page_table[row], c.lens[row], c.refs, c.lens[row], self._status,
                            c.codes, c.scales)
        if int(self._status):
            raise RuntimeError(f"a prompt of {n} tokens does not fit the cache")
        return int(e.tokens[0])

    # -- speculative decoding -------------------------------------------------------------------
    def verify(self, tokens, parents):
        """tokens, parents int32 [slots, nodes] (device): the model's predictions after each node,
        int32 [slots, nodes]; `logits` holds the rows. The nodes' keys and values are kept
        for `accept`. Nothing waits for the GPU; `check` does, and raises if the attention gave up."""
        c, B, N = self.cache, self.slots, self.nodes
        G, D = self.s.n_kv_groups, self.s.head_dim
        depth = torch.zeros(B, N, **self._ints)
        up = parents.clone()
        for _ in range(N):  # a node's depth: how often its parent has one
            depth += up >= 0
            up = torch.where(up >= 0, torch.gather(parents, 1, up.clamp(0, N - 1).long()), up)
        positions = self._in_table(c.lens[:, None] + depth).reshape(-1).contiguous()

        def attend(li, q, k, v, out):
            self._k[li].copy_(k.view(B, N, G, D))
            self._v[li].copy_(v.view(B, N, G, D))
            self._tree(q.view(B, N, -1, D), self._k[li], self._v[li], c.k[li], c.v[li], c.page_table, c.lens, parents,
                       out.view(B, N, -1, D))

        return self._forward(tokens.reshape(-1), positions, attend).view(B, N)

    def check(self):
        """Waits for the GPU and raises RuntimeError if the cache refused a slot or a tree attention
        gave up a bounded wait since the last check."""
        TreeAttention.check()
        self.cache.check()

    def accept(self, paths):
        """Appends the listed nodes of the last `verify` to their slots (an empty list: none)."""
        index = torch.tensor([p + [-1] * (self.nodes - len(p)) for p in paths], dtype=torch.int32)
        self.cache.append(self._k, self._v, index.to(self.engine.dev))

    def generate(self, prompts, max_new: int, stop: int | None = None):
        """Greedy continuations (lists of max_new tokens, or up to `stop`) of at most `slots`
        prompts, decoded speculatively. Finished slots are freed. A prompt and its continuation need
        room for all their tokens but the last; RuntimeError if the cache refuses a slot."""
        if not 1 <= len(prompts) <= self.slots:
            raise ValueError(f"generate takes 1 to {self.slots} prompts, got {len(prompts)}")
        self.cache.check()  # a refusal from before is not this one's
        dev, N = self.engine.dev, self.nodes
        self.cache.free(range(self.slots))
        texts = [list(p) for p in prompts]
        done = [False] * len(texts)
        for i, t in enumerate(texts):
            t.append(self.prefill(t, i))
        self.passes = 0
        while True:
            for i, (t, p) in enumerate(zip(texts, prompts)):
                if not done[i] and (len(t) - len(p) >= max_new or t[-1] == stop):
                    done[i] = True
                    self.cache.free([i])
            if all(done):
                return [t[len(p) : len(p) + max_new] for t, p in zip(texts, prompts)]
            drafts = [lookup_draft(t, N) if not d else ([0] * N, [-2] * N) for t, d in zip(texts, done)]
            drafts += [([0] * N, [-2] * N)] * (self.slots - len(texts))
            tokens, parents = (torch.tensor([d[i] for d in drafts], dtype=torch.int32, device=dev) for i in (0, 1))
            predicted = self.verify(tokens, parents).tolist()
            TreeAttention.check()
            self.passes += 1
            paths, more = [[] for _ in range(self.slots)], [[] for _ in texts]
            for i, (t, p) in enumerate(zip(texts, prompts)):
                if done[i]:
                    continue
                path = accepted_path(*drafts[i], predicted[i])
                left = max_new - (len(t) - len(p))
                more[i] = [predicted[i][n] for n in path][:left]
                if stop in more[i]:
                    more[i] = more[i][: more[i].index(stop) + 1]
                if len(more[i]) < left and more[i][-1] != stop:
                    paths[i] = path  # the slot goes on: the next pass reads these rows
            if any(paths):
                self.accept(paths)
                self.cache.check()
            for t, new in zip(texts, more):
                t.extend(new)

    # -- long contexts -----------------------------------------------------------------------------
    def decode_selected(self, tokens):
        """One token per slot (int32 [slots], device), read through the selected pages: appends
        its keys and values and returns the predictions, int32 [slots]. Every slot takes part: if
        the cache refuses one, RuntimeError, and all keep their lengths."""
        c, B = self.cache, self.slots
        index = torch.zeros(B, 1, **self._ints)
        after = c.lens + 1
        before, positions = c.lens.clone(), self._in_table(c.lens)
        last = self.s.n_layers - 1
        refused = torch.zeros_like(self._status)

        def attend(li, q, k, v, out):
            # the page table is extended by the first layer; the lengths move with the last one
            layer = slice(li, li + 1)
            lens_out = c.lens if li == last else self._scratch
            self._layer_append(k.contiguous().view(1, B, 1, *k.shape[1:]), v.contiguous().view(1, B, 1, *v.shape[1:]), index,
                               c.k[layer], c.v[layer], c.page_table, c.lens, c.refs, lens_out, self._status,
                               c.codes[layer], c.scales[layer])
            if li == 0:
                refused.copy_(self._status)
            self._select(q, *c.layer(li), c.page_table, after, out, self.selected)

        out = self._forward(tokens, positions, attend)
        if int(refused):
            c.lens.copy_(before)  # the others' rows are written again when the step is repeated
            raise RuntimeError("a slot was refused: no free page, a full table row, or a shared page to be written")
        return out
