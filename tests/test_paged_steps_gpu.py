"""Steps of the paged cache as a program mixes them: prompts admitted eagerly with counts from the host or the device
between replays of a captured decode step, attention into buffers of its own, steps that refuse requests."""

import ctypes

import numpy as np
import pytest

from oracle import paged as P
from torchnative_amd.tensor import current_stream

pytestmark = pytest.mark.gpu

N, H, G, D, S, WIDTH, PAGES, TOKENS = 4, 2, 3, 64, 16, 8, 24, 96
MOST = WIDTH * S


@pytest.fixture(scope="module")
def tn():
    import torchnative_amd as tn

    return tn


class Loop:
    """A table, a cache and the step's inputs, and the oracle's beside them."""

    def __init__(self, tn, seed=0):
        self.tn, self.rng = tn, np.random.default_rng(seed)
        self.table, self.dev = tn.PageTable(N, WIDTH, S, PAGES, TOKENS), tn.Q4Cache(PAGES, S, H, D)
        self.k, self.v = (tn.zeros((TOKENS, H, D)) for _ in "kv")
        self.q = tn.zeros((TOKENS, H * G, D))
        self.cache = P.Cache(PAGES, S, H, D)
        self.o = {"lens": np.zeros(N, np.int32), "table": np.full((N, WIDTH), -1, np.int32),
                  "free": np.arange(PAGES, dtype=np.int32)[::-1].copy(), "state": np.array([PAGES, 0], np.int32)}

    def write(self, t, a):
        from torchnative_amd import _lib as L

        a = np.ascontiguousarray(a)
        L.check(L.lib().tn_memcpy_h2d(t.data_ptr(), a.ctypes.data, a.nbytes, current_stream()))

    def inputs(self):
        self.kv = [self.rng.standard_normal((TOKENS, H, D)).astype(np.float32) for _ in "kv"]
        self.qq = self.rng.standard_normal((TOKENS, H * G, D)).astype(np.float32)
        for t, a in zip((self.k, self.v, self.q), (*self.kv, self.qq)):
            self.write(t, a)

    def check(self, fresh, out, lse, note):
        fresh = np.asarray(fresh, np.int32)
        o = self.o = P.plan(fresh, self.o["lens"], self.o["table"], S, self.o["free"], self.o["state"], TOKENS)
        self.cache.append(*self.kv, o["slots"])
        t = self.table
        assert np.array_equal(t.fresh.numpy(), fresh), note
        for name in ("lens", "base", "state", "row_start", "slots", "pos"):
            got = getattr(t, name).numpy()
            assert np.array_equal(got, o[name]), f"{note} {name}: {got} {o[name]}"
        ref = P.attend(self.qq.astype(np.float64), self.cache, o["row_start"], o["lens"], o["table"])
        tol, ltol = P.tolerance("float32", np.nan_to_num(ref[0]), ref[1], *(np.nan_to_num(x) for x in ref[2:]), MOST, D)
        live = o["slots"] >= 0
        assert live.any(), note
        assert (np.abs(out.numpy()[live] - ref[0][live]) <= tol[live]).all(), note
        assert (np.abs(lse.numpy()[live] - ref[1][live]) <= ltol[live]).all(), note
        return ref


def test_eager_admissions_between_replays_of_a_captured_step(tn):
    from torchnative_amd import _lib as L

    lib, s = L.lib(), tn.Stream()
    with s:
        w = Loop(tn)
        t = w.table
        out, lse = tn.zeros((TOKENS, H * G, D)), tn.zeros((TOKENS, H * G))
        work = tn.empty((w.dev.work_floats(N, TOKENS, H * G, TOKENS, MOST) + 1,), "float32", "hip")
        held = t.fresh.data_ptr()
        L.check(lib.tn_stream_begin_capture(s.handle))
        t.step()
        w.dev.append(w.k, w.v, t.slots)
        w.dev.attend(w.q, t, TOKENS, MOST, work=work, out=out, lse=lse)
        graph = ctypes.c_void_p()
        L.check(lib.tn_stream_end_capture(s.handle, ctypes.byref(graph)))

        ones = [1, 1, 0, 0]
        for i, (how, fresh) in enumerate([
                ("host", [40, 3, 0, 0]), ("replay", ones), ("replay", ones), ("device", [0, 0, 33, 0]),
                ("replay", [1, 1, 1, 0]), ("host", [1, -1, 1, 50]), ("replay", [1, 0, 1, 1]), ("again", [1, 0, 1, 1]),
                ("device", [-1, 9, 1, 1]), ("again", [-1, 9, 1, 1]), ("replay", [0, 1, 1, 1]), ("host", (7, 1, 1, 1)),
                ("replay", [1, 1, 1, 1])]):
            w.inputs()
            if how == "replay":
                w.write(t.fresh, np.asarray(fresh, np.int32))
                L.check(lib.tn_graph_launch(s.handle, graph))
                got = out, lse
            else:
                if how == "again":
                    t.step()
                elif how == "host":
                    t.step(fresh)
                else:  # a tensor of the caller's, gone when the call returns
                    t.step(tn.tensor(np.asarray(fresh, np.int32), device="hip"))
                w.dev.append(w.k, w.v, t.slots)
                got = w.dev.attend(w.q, t, TOKENS, MOST)
            s.synchronize()
            w.check(fresh, *got, f"step {i}, {how}")
            assert t.fresh.data_ptr() == held
        L.check(lib.tn_graph_destroy(graph))
