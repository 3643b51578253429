"""A key/value cache in pages, held in 4 bits, and the attention over it.

The serving counterpart of the reference's per-sequence `PreallocatedLayer`
(torchnative/python/torchnative/kernels/kv_cache.py:92-114): the sequences of a
batch share one pool of pages (`Q4Cache`, one a layer), a device-resident
`PageTable` hands pages to requests and gives each new token its slot, and
`Q4Cache.attend` runs the rows of all requests, single tokens and prompts alike,
over what they have cached.

    pages = PageTable(requests=16, width=256, page_size=16, pages=4096, tokens=512)
    cache = Q4Cache(4096, 16, n_kv_heads, head_dim)
    pages.step(fresh)                         # int32 [16]: new tokens of each request, -1: ended
    cache.append(k, v, pages.slots)           # [512, n_kv_heads, head_dim]
    out, lse = cache.attend(q, pages, max_rows, max_len)

Everything a step needs lies on the device, so a decode loop can be captured
once and replayed. Tensors off the hip device are refused.
"""

from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._C import _dt, _require_hip
from ._lib import check, lib
from .tensor import Tensor, current_stream, tensor

__all__ = ["PageTable", "Q4Cache"]


def _int32(op, **named):
    for name, t in named.items():
        if t.dtype != "int32":
            raise NotImplementedError(f"{op}: {name} must be int32, got {t.dtype}")


class PageTable:
    """The pages of `requests` slots, at most `width` each, out of a pool of `pages`; a step has at most `tokens`
    rows. `lens`, `row_start`, `base`, `slots`, `pos`, `table` and `state` are device int32 tensors that `step`
    updates in place (include/tnhip.h, tn_paged_plan). A request whose tokens do not fit is refused: `base` -1, its rows'
    `slots` -1, its length as it was; `state[1]` is 0 where none was."""

    def __init__(self, requests: int, width: int, page_size: int, pages: int, tokens: int):
        self.requests, self.width, self.page_size = int(requests), int(width), int(page_size)
        self.pages, self.tokens = int(pages), int(tokens)

        def ints(*shape, fill=0):
            return tensor(np.full(shape, fill, np.int32), device="hip")

        self.fresh, self.lens, self.base = ints(requests), ints(requests), ints(requests)
        self.table = ints(requests, width, fill=-1)
        # popped from the end: page 0 goes first
        self.free_pages = tensor(np.arange(pages, dtype=np.int32)[::-1].copy(), device="hip")
        self.state = tensor(np.array([pages, 0], np.int32), device="hip")
        self.row_start = ints(requests + 1)
        self.slots, self.pos = ints(tokens, fill=-1), ints(tokens)

    def step(self, fresh=None) -> None:
        """Adds fresh[r] tokens to request r, or ends it (negative). `fresh` is a device int32 tensor or host numbers,
        copied into `self.fresh`, or None for `self.fresh` as it stands (a captured loop writes it on the device).
        `self.fresh` is one buffer for the table's life: captured steps hold its address. Host numbers wait for the
        stream and cannot be captured."""
        op = "paged_plan"
        own = self.fresh
        if fresh is not None:
            given = fresh if isinstance(fresh, Tensor) else np.ascontiguousarray(fresh, np.int32)
            if isinstance(given, Tensor):
                _require_hip(op, given)
                _int32(op, fresh=given)
            if np.shape(fresh) != own.shape:
                raise RuntimeError(
                    f"{op}: fresh {list(np.shape(fresh))} does not give {self.requests} requests a count each")
            if not isinstance(given, Tensor):
                check(lib().tn_memcpy_h2d(own.data_ptr(), given.ctypes.data, own.nbytes, current_stream()))
            elif given.data_ptr() != own.data_ptr():
                check(lib().tn_memcpy_d2d(own.data_ptr(), given.data_ptr(), own.nbytes, current_stream()))
        check(lib().tn_paged_plan(
            current_stream(), self.requests, own.data_ptr(), self.lens.data_ptr(), self.lens.data_ptr(),
            self.table.data_ptr(), self.width, self.page_size, self.free_pages.data_ptr(), self.pages,
            self.state.data_ptr(), self.state.data_ptr(), self.tokens, self.row_start.data_ptr(),
            self.base.data_ptr(), self.slots.data_ptr(), self.pos.data_ptr()))


class Q4Cache:
    """One layer's keys and values in pages of q4_0 blocks (include/tnhip.h, tn_q4_cache): page_size a power of two
    from 16 to 256, head_dim a multiple of 32 up to 256."""

    def __init__(self, pages: int, page_size: int, n_kv_heads: int, head_dim: int):
        self.pages, self.page_size = int(pages), int(page_size)
        self.n_kv_heads, self.head_dim = int(n_kv_heads), int(head_dim)
        rows = self.pages * self.n_kv_heads * self.page_size
        self.k_codes, self.v_codes = (Tensor((rows * self.head_dim // 2,), "uint8", "hip") for _ in range(2))
        self.k_scales, self.v_scales = (Tensor((rows * (self.head_dim // 32),), "float16", "hip") for _ in range(2))
        self._c = _lib.Q4Cache(self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(),
                               self.v_scales.data_ptr(), self.pages, self.page_size, self.n_kv_heads, self.head_dim)
        self._work = {}

    def _ref(self):
        return ctypes.byref(self._c)

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales))

    def _rows(self, op, t):
        if t.dim() != 3 or t.shape[1:] != (self.n_kv_heads, self.head_dim):
            raise RuntimeError(f"{op}: rows {list(t.shape)} are not [m, {self.n_kv_heads}, {self.head_dim}]")

    def append(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Writes rows k, v [m, n_kv_heads, head_dim] to `slots` [m]; a negative slot skips its row."""
        op = "kv_append_q4_0"
        _require_hip(op, k, v, slots)
        _int32(op, slots=slots)
        self._rows(op, k)
        if v.shape != k.shape or v.dtype != k.dtype or slots.shape != k.shape[:1]:
            raise RuntimeError(f"{op}: k {list(k.shape)} {k.dtype}, v {list(v.shape)} {v.dtype} and slots "
                               f"{list(slots.shape)} do not describe one set of rows")
        check(lib().tn_kv_append_q4_0(current_stream(), self._ref(), _dt(k.dtype), k.data_ptr(), v.data_ptr(),
                                      k.shape[0], self.n_kv_heads * self.head_dim, slots.data_ptr()))

    def read(self, slots: Tensor, dtype: str = "float32"):
        """The cached rows at `slots` [m], as (k, v) [m, n_kv_heads, head_dim]."""
        op = "kv_read_q4_0"
        _require_hip(op, slots)
        _int32(op, slots=slots)
        k, v = (Tensor((slots.numel, self.n_kv_heads, self.head_dim), dtype, "hip") for _ in range(2))
        check(lib().tn_kv_read_q4_0(current_stream(), self._ref(), slots.data_ptr(), slots.numel, _dt(dtype),
                                    k.data_ptr(), v.data_ptr()))
        return k, v

    def work_floats(self, requests: int, tokens: int, heads: int, max_rows: int, max_len: int) -> int:
        """Floats of scratch that `attend` takes for such a call."""
        return int(lib().tn_sdpa_paged_q4_0_work_floats(self._ref(), requests, tokens, heads, max_rows, max_len))

    def attend(self, q: Tensor, pages: PageTable, max_rows: int, max_len: int, scale: float | None = None,
               work: Tensor | None = None, out: Tensor | None = None, lse: Tensor | None = None):
        """The rows q [tokens, heads, head_dim] of `pages`' last step over their requests' cached tokens, the rows'
        own among them. max_rows, max_len: upper bounds of a request's rows and length. Returns (out, lse), whose rows
        behind the last request's are left as they were.
        Rows of a request that the step refused (`pages.base` -1, `pages.slots` -1) are not in the cache; what they get
        here is the attention of the request's earlier tokens, to be dropped.

        `work`, `out` and `lse` are made where they are not given. Code that captures passes its own, so that the
        graph's buffers live as long as it does, a `work` of its own for each graph."""
        op = "sdpa_paged_q4_0"
        _require_hip(op, q)
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise RuntimeError(f"{op}: query {list(q.shape)} is not [tokens, heads, {self.head_dim}]")
        if pages.page_size != self.page_size:
            raise RuntimeError(f"{op}: the table's pages hold {pages.page_size} tokens, the cache's {self.page_size}")
        T, Hq, D = q.shape
        need = self.work_floats(pages.requests, T, Hq, max_rows, max_len)
        if work is None:  # one a stream: calls on a stream are ordered
            held = self._work.setdefault(current_stream(), [])  # outgrown ones stay: a graph may point at them
            if not held or held[-1].numel < need:
                held.append(Tensor((max(need, 2 * held[-1].numel if held else 1),), "float32", "hip"))
            work = held[-1]
        out = Tensor(q.shape, q.dtype, "hip") if out is None else out
        lse = Tensor((T, Hq), "float32", "hip") if lse is None else lse
        _require_hip(op, work, out, lse)
        if (out.shape, out.dtype, lse.shape, lse.dtype, work.dtype) != (q.shape, q.dtype, (T, Hq), "float32", "float32"):
            raise RuntimeError(f"{op}: out {list(out.shape)} {out.dtype}, lse {list(lse.shape)} {lse.dtype} or work "
                               f"{work.dtype} does not fit query {list(q.shape)} {q.dtype}")
        sc = float("nan") if scale is None else float(scale)
        check(lib().tn_sdpa_paged_q4_0(
            current_stream(), self._ref(), _dt(q.dtype), q.data_ptr(), Hq * D, T, Hq, pages.requests,
            pages.row_start.data_ptr(), pages.lens.data_ptr(), pages.table.data_ptr(), pages.width, max_rows, max_len,
            sc, work.data_ptr(), work.numel, out.data_ptr(), lse.data_ptr()))
        return out, lse
