"""PageTable's buffers off the GPU, over a stand-in for the library that keeps device memory in host buffers: a captured
step holds the addresses that the table had when it was captured, so no later step may replace or free them."""

import ctypes
import gc

import numpy as np
import pytest

from torchnative_amd import _lib
from torchnative_amd.paged import PageTable
from torchnative_amd.tensor import tensor


class HostLibrary:
    """Allocation and copies in host memory; tn_paged_plan notes its arguments and the counts it would read."""

    def __init__(self):
        self.live, self.plans, self.streams = {}, [], []

    def tn_malloc(self, out, nbytes):
        b = ctypes.create_string_buffer(max(nbytes, 1))
        self.live[ctypes.addressof(b)] = b
        out._obj.value = ctypes.addressof(b)
        return _lib.TN_OK

    def tn_free(self, ptr):
        self.live.pop(ptr, None)
        return _lib.TN_OK

    def _copy(self, dst, src, nbytes, stream):
        ctypes.memmove(dst, src, nbytes)
        self.streams.append(stream)
        return _lib.TN_OK

    tn_memcpy_h2d = tn_memcpy_d2h = tn_memcpy_d2d = _copy

    def tn_paged_plan(self, stream, n, fresh, *rest):
        assert fresh in self.live, "the counts were freed"
        self.plans.append((stream, fresh, *rest))
        return list((ctypes.c_int32 * n).from_address(fresh)) and _lib.TN_OK

    def counts(self, call):
        """What call number `call` reads now: a replay of it."""
        fresh = self.plans[call][1]
        assert fresh in self.live, "a replay would read freed memory"
        return list((ctypes.c_int32 * 3).from_address(fresh))


@pytest.fixture
def host(monkeypatch):
    h = HostLibrary()
    monkeypatch.setattr(_lib, "_lib", h)
    yield h
    gc.collect()  # what the test allocated goes back to the stand-in


def _table():
    return PageTable(requests=3, width=4, page_size=16, pages=12, tokens=48)


@pytest.mark.parametrize("give", [lambda x: x, np.array, lambda x: np.array(x, np.int64)[::1], tuple,
                                  lambda x: tensor(np.array(x, np.int32), device="hip")])
def test_a_step_with_counts_keeps_the_buffer_that_a_captured_step_reads(host, give):
    t = _table()
    at = t.fresh.data_ptr()
    t.step()  # what a graph would hold
    t.step(give([5, -1, 7]))
    gc.collect()
    assert t.fresh.data_ptr() == at and host.plans[1][1] == at
    assert host.counts(0) == [5, -1, 7]
    t.step()  # the counts stand
    assert host.counts(2) == [5, -1, 7] and host.plans[2] == host.plans[0]
    assert set(host.live) >= {x for x in host.plans[0][2:] if isinstance(x, int) and x > 1 << 16}


def test_the_callers_tensor_is_not_the_tables(host):
    t = _table()
    mine = tensor(np.array([1, 2, 3], np.int32), device="hip")
    t.step(mine)
    _lib.lib().tn_memcpy_h2d(mine.data_ptr(), (ctypes.c_int32 * 3)(9, 9, 9), 12, None)
    assert t.fresh.data_ptr() != mine.data_ptr() and host.counts(0) == [1, 2, 3]
    t.step(t.fresh)  # its own, and a view of it
    t.step(t.fresh.view(3))
    assert host.counts(2) == [1, 2, 3]


def test_counts_that_do_not_fit_are_refused_before_anything_is_copied(host):
    t = _table()
    n = len(host.streams)
    for bad in ([1, 2], [[1, 2, 3]], 4, tensor(np.zeros(2, np.int32), device="hip")):
        with pytest.raises(RuntimeError, match="does not give 3 requests a count each"):
            t.step(bad)
    with pytest.raises(NotImplementedError, match="fresh must be int32"):
        t.step(tensor(np.zeros(3, np.float32), device="hip"))
    with pytest.raises(NotImplementedError, match="device"):
        t.step(tensor(np.zeros(3, np.int32), device="cpu"))
    assert not host.plans and len(host.streams) == n + 2  # the two tensors of the test
