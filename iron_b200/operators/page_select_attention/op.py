"""Decode attention over the pages of a paged KV cache that a cheap score selects.

Over a long context a query reads only ``top_pages`` pages per kv head: the last page, the
first one, and the pages whose summary (PageAppend keeps it) bounds the query group's logits
highest. The score is a sum of whole numbers times one scale, so the selection does not
depend on any order of summation; of equal scores the lower page wins. The exact rule is
that of ``iron_page_select_attn`` in include/iron_b200.h. IRON has no counterpart; with every
page selected this is its decode attention (iron/applications/llama_3.2_1b/
llama_npu.py:495-529).

Buffers: q bf16 [batch, num_heads, head_dim] (may be a strided view); k_pages, v_pages bf16
[num_pages, num_kv_heads, page_size, head_dim], codes int8 [num_pages, num_kv_heads, 2,
head_dim], scales fp32 [num_pages, num_kv_heads] (one layer of the pool); page_table int32
[batch, max_pages]; lens int32 [batch] (tokens, the current one included); out bf16 like q;
selected int32 [batch, num_kv_heads, top_pages]: the pages' places in the sequence,
ascending, then -1.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field

import numpy as np

from ... import _lib
from ...common.base import AIERuntimeArgSpec
from ...common.paged import PagedOperator, address, stride_array
from ...common.verify import Tolerance


@dataclass
class PageSelectAttention(PagedOperator):
    batch: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    max_pages: int
    top_pages: int
    scale: float | None = None
    context: object = field(default=None, repr=False)

    _tolerance = Tolerance.relative(2e-2, 1e-2)
    _strided = (0, 7)

    def __post_init__(self):
        if not 1 <= self.batch <= 65535:
            raise ValueError(f"batch must be 1 to 65535, got {self.batch}")
        if not 1 <= self.top_pages <= 4096:
            raise ValueError(f"top_pages must be 1 to 4096, got {self.top_pages}")
        if self.num_kv_heads < 1 or self.num_heads % self.num_kv_heads or not 1 <= self.num_heads // self.num_kv_heads <= 16:
            raise ValueError("num_heads must be a multiple of num_kv_heads (group <= 16)")
        self._check_geometry()
        PagedOperator.__init__(self, context=self.context)

    def get_arg_spec(self):
        B, G, D = self.batch, self.num_kv_heads, self.head_dim
        pages = (self.num_pages, G, self.page_size, D)
        spec = AIERuntimeArgSpec
        return [spec("in", (B, self.num_heads, D)), spec("in", pages), spec("in", pages),
                spec("in", (self.num_pages, G, 2, D), dtype=np.int8), spec("in", (self.num_pages, G), dtype=np.float32),
                spec("in", (B, self.max_pages), dtype=np.int32), spec("in", (B,), dtype=np.int32),
                spec("out", (B, self.num_heads, D)), spec("out", (B, G, self.top_pages), dtype=np.int32)]

    def workspace_bytes(self) -> int:
        return _lib.load().iron_page_select_attn_workspace_bytes(
            self.batch, self.num_heads, self.num_kv_heads, self.head_dim, self.max_pages, self.top_pages, self.page_size)

    def _launch(self, q, k_pages, v_pages, codes, scales, page_table, lens, out, selected, *, stream, flags=0):
        p = address
        rows = (self.batch, self.num_heads, self.head_dim)
        ws, nbytes = self._workspace(stream)
        pool = _lib.PagePool(p(k_pages), p(v_pages), p(codes), p(scales), p(page_table), p(lens), None, 1, self.batch,
                             self.num_pages, self.max_pages, self.num_kv_heads, self.head_dim, self.page_size)
        scale = 1.0 / math.sqrt(self.head_dim) if self.scale is None else self.scale
        _lib.call("iron_page_select_attn", ctypes.byref(pool), p(q), p(out), p(selected), self.num_heads,
                  self.top_pages, stride_array(q, rows), stride_array(out, rows), scale, ws, nbytes, flags, stream)

    def reference(self, q, k_pages, v_pages, codes, scales, page_table, lens):
        """(out, selected) by the rule, head by head."""
        import torch

        g, D = self.num_heads // self.num_kv_heads, self.head_dim
        scale = 1.0 / math.sqrt(D) if self.scale is None else self.scale
        out = torch.zeros(self.batch, self.num_heads, D)
        selected = torch.full((self.batch, self.num_kv_heads, self.top_pages), -1, dtype=torch.int32)
        for b in range(self.batch):
            L = int(lens[b])
            n = -(-L // self.page_size)
            if n == 0:
                continue
            ids = page_table[b, :n].long()
            for h in range(self.num_kv_heads):
                x = q[b, h * g : h * g + g].float()
                a = x.abs().max()
                q8 = torch.round(x / a * 127.0).long() if 0 < float(a) < math.inf else torch.zeros_like(x).long()
                lo, hi = codes[ids, h, 0].long(), codes[ids, h, 1].long()
                score = (q8[:, None].clamp(min=0) * hi + q8[:, None].clamp(max=0) * lo).sum((0, 2)).float() * scales[ids, h]
                score = score.clamp(-3.4028234663852886e38, 3.4028234663852886e38).tolist()
                order = sorted(range(1, n - 1), key=lambda i: (-score[i], i))
                keep = sorted(([n - 1] + ([0] if n > 1 else []) + order)[: self.top_pages])
                selected[b, h, : len(keep)] = torch.tensor(keep, dtype=torch.int32)
                t = torch.cat([torch.arange(i * self.page_size, min(L, (i + 1) * self.page_size)) for i in keep])
                at, r = ids[t // self.page_size], t % self.page_size
                s = (x @ k_pages[at, h, r].float().T) * scale
                out[b, h * g : h * g + g] = torch.softmax(s, -1) @ v_pages[at, h, r].float()
        return out.to(torch.bfloat16), selected
