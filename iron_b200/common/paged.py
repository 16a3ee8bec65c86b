"""Base of the operators on a paged KV cache.

IRON's cache is one padded buffer per sequence (iron/applications/llama_3.2_1b/
llama_npu.py:481-495); pages of a shared pool have no counterpart there. The layout is
that of ``iron_page_pool`` in include/iron_b200.h:

- ``k_pool``, ``v_pool`` bf16 [layers, pages, kv_heads, page_size, head_dim];
- ``codes`` int8 [layers, pages, kv_heads, 2, head_dim], ``scales`` fp32 [layers, pages,
  kv_heads]: the summaries of full pages that PageSelectAttention scores;
- ``page_table`` int32 [slots, max_pages] (-1: no page), ``lens`` int32 [slots], ``refs``
  int32 [pages].
"""

from __future__ import annotations

import ctypes

import numpy as np

from .. import _lib
from .base import MLIROperator
from .tensor import np_dtype

PAGE_SIZES = (16, 32, 64, 128)


class PagedOperator(MLIROperator):
    """Checks each buffer's device, type, size and order, and keeps one workspace per device and
    stream (calls on different streams may overlap; calls on one stream follow one another).

    A CUDA graph may replay on any stream, beside anything, so the calls that it captures have a
    workspace of the graph's own (one per captured stream), taken from the graph's memory."""

    def _check_geometry(self):
        if self.head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {self.head_dim}")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {self.page_size}")
        for name in ("num_pages", "max_pages", "num_kv_heads"):
            if getattr(self, name) < 1:
                raise ValueError(f"{name} must be positive, got {getattr(self, name)}")
        if self.max_pages * self.page_size > (1 << 31) - 128:
            raise ValueError("max_pages * page_size must be at most 2^31 - 128 tokens")
        import torch

        self._spaces = {}
        self._captured = {}
        self._wanted = None
        self._device, self._capturing = torch.cuda.current_device, torch.cuda.is_current_stream_capturing

    def workspace_bytes(self) -> int:
        raise NotImplementedError

    def share_workspaces(self, other: "PagedOperator"):
        """Calls of this operator use the workspaces of `other`, whose size must do for both, and
        must not overlap its calls on the same stream. Returns self."""
        self._spaces = other._spaces
        return self

    def counter_bytes(self) -> int:
        """Bytes at the start of the workspace that must be zero before its first use."""
        return 0

    def _workspace(self, stream: int):
        """(address, bytes) of the workspace of this stream, or of the graph that it captures."""
        if self._capturing():
            return self._graph_workspace(stream)
        if self._captured:  # the graph keeps the memory, and sets it up again in each replay
            self._captured = {}
        key = self._device(), stream
        ws = self._spaces.get(key)
        if ws is None:
            import torch

            t = torch.zeros(max(16, self.workspace_bytes()), dtype=torch.uint8, device="cuda")
            ws = self._spaces[key] = (t.data_ptr(), t.numel(), t)
        return ws[0], ws[1]

    def _graph_workspace(self, stream: int):
        import torch

        capture = ctypes.c_uint64()
        _lib.call("iron_capture_id", stream, ctypes.byref(capture))
        key = capture.value, stream
        ws = self._captured.get(key)
        if ws is None:
            t = torch.empty(max(16, self.workspace_bytes()), dtype=torch.uint8, device="cuda")
            if self.counter_bytes():
                t[: self.counter_bytes()].zero_()  # part of the graph
            ws = (t.data_ptr(), t.numel(), t)
            self._captured = {k: w for k, w in self._captured.items() if k[0] == key[0]} | {key: ws}
        return ws[0], ws[1]

    def prepare(self):
        self._workspace(_lib.current_stream())

    # buffers that may be views with strides (last dimension contiguous)
    _strided: tuple = ()

    def _check_buffers(self, bufs) -> None:
        import torch

        if self._wanted is None:
            kinds = {np.dtype(np.int32): torch.int32, np.dtype(np.int8): torch.int8, np.dtype(np.float32): torch.float32}
            self._wanted = [(kinds.get(np.dtype(np_dtype(s.dtype)), torch.bfloat16), int(np.prod(s.shape, dtype=np.int64)),
                             s.shape if i in self._strided else None) for i, s in enumerate(self.get_arg_spec())]
        if len(bufs) != len(self._wanted):
            raise ValueError(f"{type(self).__name__} takes {len(self._wanted)} buffers, got {len(bufs)}")
        for t, (dtype, numel, view) in zip(bufs, self._wanted):
            if t.dtype is not dtype or not (t.numel() >= numel if t.is_contiguous() else
                                            view and t.shape == view and t.stride(-1) == 1):
                self._refuse_buffers(bufs)

    def _refuse_device(self, bufs, device):
        for i, t in enumerate(bufs):
            if address(t) and t.get_device() != device:
                raise ValueError(f"buffer {i} of {type(self).__name__} is on {t.device}, the current device is {device}")

    def _refuse_buffers(self, bufs):
        """Raises for what is wrong with the buffers."""
        me = type(self).__name__
        for i, (t, (dtype, numel, view)) in enumerate(zip(bufs, self._wanted)):
            if t.dtype is not dtype:
                raise ValueError(f"buffer {i} of {me} is {t.dtype}, needs {dtype}")
            if t.is_contiguous():
                if t.numel() < numel:
                    raise ValueError(f"buffer {i} of {me} holds {t.numel()} values, needs {numel}")
            elif view is None or t.shape != view:
                raise ValueError(f"buffer {i} of {me} must be contiguous")
            elif t.stride(-1) != 1:
                raise ValueError(f"buffer {i} of {me} needs a contiguous last dimension")

    def get_callable(self):
        import torch

        _lib.load()
        written = [i for i, s in enumerate(self.get_arg_spec()) if s.direction != "in"]
        check, refuse, launch, device = self._check_buffers, self._refuse_device, self._launch, torch.cuda.current_device
        several = torch.cuda.device_count() > 1
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)

        def call(*bufs):
            tensors = [getattr(b, "device_tensor", b) for b in bufs]
            check(tensors)
            at = device()
            if several:
                refuse(tensors, at)
            launch(*tensors, stream=raw(at))
            for i in written:
                if bufs[i] is not tensors[i]:
                    bufs[i].mark_device_written()

        return call


def address(t):
    """Device address of a CUDA tensor."""
    if not t.is_cuda:
        raise RuntimeError("iron_b200 kernels take CUDA tensors; got a host tensor")
    return t.data_ptr()


_stride_arrays: dict = {}


def stride_array(t, shape):
    """Element strides of the leading dimensions of `t` seen as `shape`, as an int64 array for
    the C entry points (made once per set of strides, so equal strides give the same array). A
    dimension of one element has stride 0: no address depends on what the tensor says there."""
    full = t.stride()
    if t.shape != shape:
        full, step = [1], 1
        for n in reversed(shape[1:]):
            step *= n
            full.append(step)
        full = tuple(reversed(full))
    a = _stride_arrays.get((full, shape))
    if a is None:
        seen = tuple(0 if n == 1 else s for n, s in zip(shape[:-1], full))
        a = _stride_arrays.setdefault(seen, (ctypes.c_int64 * len(seen))(*seen))
        _stride_arrays[full, shape] = a
    return a
