"""Pages of a KV cache: append, fork, compact, and the cache that holds them.

IRON grows one padded buffer per sequence with StridedCopy (iron/operators/strided_copy/
op.py:18-100); a pool of pages that sequences share has no counterpart there. The rules --
which free page goes to whom, who keeps a partial page, what is refused -- are those of
``iron_page_append``, ``iron_page_fork`` and ``iron_page_compact`` in include/iron_b200.h.
Everything stays on the device: no operator waits for the host, and all can be captured in
a CUDA graph.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import numpy as np

from ... import _lib
from ...common.base import AIERuntimeArgSpec
from ...common.paged import PagedOperator, address


@dataclass
class _PoolOperator(PagedOperator):
    slots: int
    num_layers: int
    num_kv_heads: int
    head_dim: int
    page_size: int
    num_pages: int
    max_pages: int

    def __post_init__(self):
        if not 1 <= self.slots <= 2048:
            raise ValueError(f"slots must be 1 to 2048, got {self.slots}")
        if self.num_layers < 1:
            raise ValueError(f"num_layers must be positive, got {self.num_layers}")
        self._check_geometry()
        PagedOperator.__init__(self, context=self.context)

    def _pool_spec(self, direction="inout"):
        return AIERuntimeArgSpec(direction, (self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim))

    def _ints(self, direction, *shape):
        return AIERuntimeArgSpec(direction, shape, dtype=np.int32)

    def _summary_specs(self):
        if not self.summaries:
            return []
        at = (self.num_layers, self.num_pages, self.num_kv_heads)
        return [AIERuntimeArgSpec("inout", (*at, 2, self.head_dim), dtype=np.int8),
                AIERuntimeArgSpec("inout", at, dtype=np.float32)]

    def _pool(self, k, v, table, lens, refs, codes=None, scales=None):
        p = address
        return _lib.PagePool(p(k), p(v), codes if codes is None else p(codes), scales if scales is None else p(scales),
                             p(table), lens if lens is None else p(lens), p(refs), self.num_layers, self.slots,
                             self.num_pages, self.max_pages, self.num_kv_heads, self.head_dim, self.page_size)


@dataclass
class PageAppend(_PoolOperator):
    """Writes new tokens' keys and values (all layers) behind each slot's cached ones.

    Buffers: k_new, v_new bf16 [num_layers, slots, num_new, num_kv_heads, head_dim]; index
    int32 [slots, num_new]: which of the new rows to append, in order, up to the first entry
    outside [0, num_new) -- the accepted path of a tree, or 0, 1, 2, ... for a prompt; k_pool,
    v_pool; page_table (pages that are missing are allocated); lens int32 [slots]; refs;
    lens_out int32 [slots] (may be lens); status int32 [1]: slots refused for want of pages,
    of room in their table row, or because they would write a shared page; with
    ``summaries`` also codes and scales (pages that become full get theirs)."""

    num_new: int = 1
    summaries: bool = False
    context: object = field(default=None, repr=False)

    def __post_init__(self):
        if self.num_new < 1:
            raise ValueError(f"num_new must be positive, got {self.num_new}")
        if self.summaries and self.num_kv_heads * self.head_dim > 51200:
            raise ValueError("with summaries num_kv_heads * head_dim must be at most 51200")
        super().__post_init__()

    def get_arg_spec(self):
        new = AIERuntimeArgSpec("in", (self.num_layers, self.slots, self.num_new, self.num_kv_heads, self.head_dim))
        S = self.slots
        return [new, new, self._ints("in", S, self.num_new), self._pool_spec(), self._pool_spec(),
                self._ints("inout", S, self.max_pages), self._ints("in", S), self._ints("inout", self.num_pages),
                self._ints("out", S), self._ints("out", 1), *self._summary_specs()]

    def workspace_bytes(self) -> int:
        return _lib.load().iron_page_append_workspace_bytes(self.slots, self.num_pages)

    def _launch(self, k_new, v_new, index, k, v, table, lens, refs, lens_out, status, *summary, stream, flags=0):
        p = address
        ws, nbytes = self._workspace(stream)
        _lib.call("iron_page_append", ctypes.byref(self._pool(k, v, table, lens, refs, *summary)), p(k_new), p(v_new),
                  p(index), self.num_new, p(lens_out), p(status), ws, nbytes, flags, stream)


@dataclass
class PageFork(_PoolOperator):
    """Gives every slot the sequence that slot ``source[slot]`` held: keeps, forks, reorders
    (beam search) and frees (-1) in one call.

    Buffers: source int32 [slots]; page_table, lens, refs; k_pool, v_pool (the partial pages
    that need a copy get one); page_table_out, lens_out, refs_out: the new state (its table
    and refs must be other buffers than the old ones); status int32 [1]: slots left empty
    for want of pages."""

    context: object = field(default=None, repr=False)

    def get_arg_spec(self):
        S, M, P = self.slots, self.max_pages, self.num_pages
        return [self._ints("in", S), self._ints("in", S, M), self._ints("in", S), self._ints("in", P),
                self._pool_spec(), self._pool_spec(), self._ints("out", S, M), self._ints("out", S),
                self._ints("out", P), self._ints("out", 1)]

    def workspace_bytes(self) -> int:
        return _lib.load().iron_page_fork_workspace_bytes(self.slots)

    def _launch(self, source, table, lens, refs, k, v, table_out, lens_out, refs_out, status, *, stream, flags=0):
        p = address
        ws, nbytes = self._workspace(stream)
        _lib.call("iron_page_fork", ctypes.byref(self._pool(k, v, table, lens, refs)), p(source), p(table_out),
                  p(lens_out), p(refs_out), p(status), ws, nbytes, flags, stream)


@dataclass
class PageCompact(_PoolOperator):
    """Moves the used pages to the front of the pool, as few as can be.

    Buffers: page_table, refs; k_pool, v_pool; page_table_out, refs_out (each may be the old
    buffer); used int32 [1]: the number of used pages, which are now 0 .. used - 1; with
    ``summaries`` also codes and scales, which move along."""

    summaries: bool = False
    context: object = field(default=None, repr=False)

    def get_arg_spec(self):
        S, M, P = self.slots, self.max_pages, self.num_pages
        return [self._ints("in", S, M), self._ints("in", P), self._pool_spec(), self._pool_spec(),
                self._ints("out", S, M), self._ints("out", P), self._ints("out", 1), *self._summary_specs()]

    def workspace_bytes(self) -> int:
        return _lib.load().iron_page_compact_workspace_bytes(self.num_pages)

    def _launch(self, table, refs, k, v, table_out, refs_out, used, *summary, stream, flags=0):
        p = address
        ws, nbytes = self._workspace(stream)
        _lib.call("iron_page_compact", ctypes.byref(self._pool(k, v, table, None, refs, *summary)), p(table_out),
                  p(refs_out), p(used), ws, nbytes, flags, stream)


class PagedKVCache:
    """The buffers of a paged KV cache and the operators on them.

    ``append``, ``fork``, ``free`` and ``compact`` change the cache on the current stream
    without waiting for the GPU; ``check`` waits and raises RuntimeError if one of them
    refused a slot. ``layer(i)`` gives the buffers that TreeAttention (k_pages, v_pages) and
    PageSelectAttention (with codes and scales) read. ``fork`` and ``free`` write a second set of
    ``page_table``, ``lens`` and ``refs`` and swap it in, so take these from the cache for each
    call; a captured graph keeps the set that it was captured with.
    """

    def __init__(self, slots: int, num_layers: int, num_kv_heads: int, head_dim: int, page_size: int, num_pages: int,
                 max_pages: int, summaries: bool = False):
        import torch

        self._sizes = dict(slots=slots, num_layers=num_layers, num_kv_heads=num_kv_heads, head_dim=head_dim,
                           page_size=page_size, num_pages=num_pages, max_pages=max_pages)
        self._fork = PageFork(**self._sizes)
        self._compact = PageCompact(**self._sizes, summaries=summaries)
        # one operator per number of new rows; their workspaces are of one size, and shared
        self._append, self._first_append = {}, PageAppend(**self._sizes, summaries=summaries)
        self.summaries = summaries
        dev = torch.device("cuda", torch.cuda.current_device())
        pool = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        ints = dict(dtype=torch.int32, device=dev)
        self.k = torch.zeros(pool, dtype=torch.bfloat16, device=dev)
        self.v = torch.zeros_like(self.k)
        self.codes = torch.zeros(*pool[:3], 2, head_dim, dtype=torch.int8, device=dev) if summaries else None
        self.scales = torch.zeros(pool[:3], dtype=torch.float32, device=dev) if summaries else None
        self.page_table = torch.full((slots, max_pages), -1, **ints)
        self.lens, self.refs = torch.zeros(slots, **ints), torch.zeros(num_pages, **ints)
        self._other = [torch.empty_like(t) for t in (self.page_table, self.lens, self.refs)]
        self._status = torch.zeros(1, **ints)
        self._refused = torch.zeros(1, **ints)
        self._used = torch.zeros(1, **ints)

    def _summary(self):
        return (self.codes, self.scales) if self.summaries else ()

    def append(self, k_new, v_new, index):
        """k_new, v_new [num_layers, slots, n, num_kv_heads, head_dim], index int32 [slots, n]."""
        n = index.shape[1]
        if n not in self._append:
            op = PageAppend(**self._sizes, num_new=n, summaries=self.summaries)
            self._append[n] = op.share_workspaces(self._first_append).get_callable()
        self._append[n](k_new, v_new, index, self.k, self.v, self.page_table, self.lens, self.refs, self.lens,
                        self._status, *self._summary())
        self._refused += self._status

    def fork(self, source):
        """source int32 [slots]: see PageFork."""
        self._fork.get_callable()(source, self.page_table, self.lens, self.refs, self.k, self.v, *self._other, self._status)
        self._other, (self.page_table, self.lens, self.refs) = [self.page_table, self.lens, self.refs], self._other
        self._refused += self._status

    def free(self, slots):
        """Frees the listed slots."""
        import torch

        source = torch.arange(self._sizes["slots"], dtype=torch.int32)
        source[torch.as_tensor(slots, dtype=torch.long)] = -1
        self.fork(source.to(self.lens.device))

    def compact(self):
        """Packs the used pages; returns the device word that holds their number."""
        self._compact.get_callable()(self.page_table, self.refs, self.k, self.v, self.page_table, self.refs, self._used,
                                     *self._summary())
        return self._used

    def check(self):
        """Waits for the GPU and raises if a slot was refused since the last check."""
        n = int(self._refused)
        if n:
            self._refused.zero_()
            raise RuntimeError(f"{n} slot(s) refused: no free page, a full table row, or a shared page to be written")

    def layer(self, i: int):
        return (self.k[i], self.v[i], self.codes[i], self.scales[i]) if self.summaries else (self.k[i], self.v[i])
