"""Attention of a tree of drafted tokens over a paged KV cache.

A speculative decoder drafts a tree of continuations of each sequence and checks all of
them in one pass: node i attends to the sequence's cached tokens and to the nodes on its
own path. IRON has no counterpart; the one-token case is the decode attention of
iron/applications/llama_3.2_1b/llama_npu.py:495-529.

Buffers: q bf16 [batch, num_nodes, num_heads, head_dim]; k_new, v_new bf16 [batch,
num_nodes, num_kv_heads, head_dim] (the drafted tokens' own keys and values, which need not
be in the cache; q, k_new, v_new and out may be strided views, e.g. of one QKV buffer);
k_pages, v_pages bf16 [num_pages, num_kv_heads, page_size, head_dim] (one layer of the
pool); page_table int32 [batch, max_pages]; lens int32 [batch]; parents int32 [batch,
num_nodes]; out bf16 like q.

parents[b, i] is -1 (a child of the cached prefix) or a node j < i. Any other value marks an
unused place; a node below an unused one is unused too. Unused rows give zeros, and nothing
that a node's path does not hold reaches its row, whatever its values.

The kernel for many rows waits with a limit; ``check`` raises if a wait ran out.
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
class TreeAttention(PagedOperator):
    batch: int
    num_nodes: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    max_pages: int
    scale: float | None = None
    context: object = field(default=None, repr=False)

    _tolerance = Tolerance.relative(2e-2, 1e-2)
    _strided = (0, 1, 2, 8)

    def __post_init__(self):
        if not 1 <= self.num_nodes <= 128:
            raise ValueError(f"num_nodes must be 1 to 128, got {self.num_nodes}")
        if not 1 <= self.batch <= 1024:
            raise ValueError(f"batch must be 1 to 1024, got {self.batch}")
        if self.num_kv_heads < 1 or self.num_heads % self.num_kv_heads or not 1 <= self.num_heads // self.num_kv_heads <= 16:
            raise ValueError("num_heads must be a multiple of num_kv_heads (group <= 16)")
        self._check_geometry()
        if self.batch * (-(-self.max_pages * self.page_size // 64) + 5) >= 1 << 31:
            raise ValueError("batch * (max_pages * page_size / 64 + 5) must be below 2^31")
        PagedOperator.__init__(self, context=self.context)

    def get_arg_spec(self):
        B, N, D = self.batch, self.num_nodes, self.head_dim
        rows, new = (B, N, self.num_heads, D), (B, N, self.num_kv_heads, D)
        pages = (self.num_pages, self.num_kv_heads, self.page_size, D)
        spec = AIERuntimeArgSpec
        return [spec("in", rows), spec("in", new), spec("in", new), spec("in", pages), spec("in", pages),
                spec("in", (B, self.max_pages), dtype=np.int32), spec("in", (B,), dtype=np.int32),
                spec("in", (B, N), dtype=np.int32), spec("out", rows)]

    def workspace_bytes(self) -> int:
        return _lib.load().iron_tree_attn_workspace_bytes(self.batch, self.num_nodes, self.num_heads,
                                                          self.num_kv_heads, self.head_dim)

    def counter_bytes(self) -> int:
        return _lib.load().iron_tree_attn_counter_bytes(self.batch, self.num_nodes, self.num_heads, self.num_kv_heads,
                                                        self.head_dim)

    def _launch(self, q, k_new, v_new, k_pages, v_pages, page_table, lens, parents, out, *, stream, flags=0):
        p = address
        new = (self.batch, self.num_nodes, self.num_kv_heads, self.head_dim)
        rows = (self.batch, self.num_nodes, self.num_heads, self.head_dim)
        ks = stride_array(k_new, new)
        if stride_array(v_new, new) is not ks:
            raise ValueError("k_new and v_new must have the same strides")
        ws, nbytes = self._workspace(stream)
        pool = _lib.PagePool(p(k_pages), p(v_pages), None, None, p(page_table), p(lens), None, 1, self.batch,
                             self.num_pages, self.max_pages, self.num_kv_heads, self.head_dim, self.page_size)
        scale = 1.0 / math.sqrt(self.head_dim) if self.scale is None else self.scale
        _lib.call("iron_tree_attn", ctypes.byref(pool), p(q), p(k_new), p(v_new), p(parents), p(out), self.num_nodes,
                  self.num_heads, stride_array(q, rows), ks, stride_array(out, rows), scale, ws,
                  nbytes, flags, stream)

    @staticmethod
    def check():
        """Waits for the GPU and raises RuntimeError if a bounded wait ran out in a tree attention
        on the current device since the last check: outputs of the calls in between are not whole."""
        status = _lib.load().iron_tree_attn_status(1)
        if status == _lib.IRON_ERR_TIMEOUT:
            raise RuntimeError("TreeAttention: a bounded wait timed out, the outputs are not whole")
        _lib.check(status, "iron_tree_attn_status")

    def reference(self, q, k_new, v_new, k_pages, v_pages, page_table, lens, parents):
        """The formula, row by row, in fp32."""
        import torch

        B, N, D = self.batch, self.num_nodes, self.head_dim
        g = self.num_heads // self.num_kv_heads
        scale = 1.0 / math.sqrt(D) if self.scale is None else self.scale
        q, k_new, v_new = (t.reshape(B, N, -1, D).float() for t in (q, k_new, v_new))
        out = torch.zeros(B, N, self.num_heads, D)
        for b in range(B):
            n = int(lens[b])
            ids = page_table[b, : -(-n // self.page_size)].long()
            K, V = (x[ids].transpose(0, 1).reshape(self.num_kv_heads, -1, D)[:, :n].float() for x in (k_pages, v_pages))
            paths = []
            for i in range(N):
                par = int(parents[b, i])
                path = [i] if par == -1 else paths[par] + [i] if 0 <= par < i and paths[par] else []
                paths.append(path)
                if not path:
                    continue
                k = torch.cat([K, k_new[b, path].transpose(0, 1)], 1).repeat_interleave(g, 0)
                v = torch.cat([V, v_new[b, path].transpose(0, 1)], 1).repeat_interleave(g, 0)
                s = torch.einsum("hd,hld->hl", q[b, i], k) * scale
                out[b, i] = torch.einsum("hl,hld->hd", torch.softmax(s, -1), v)
        return out.to(torch.bfloat16)
