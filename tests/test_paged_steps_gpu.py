"""Steps of the paged cache as a program mixes them: prompts admitted eagerly with counts from the host or the device
between replays of a captured decode step, attention into buffers of its own, steps that refuse requests."""

import ctypes

import numpy as np
import pytest

from oracle import paged as P
from test_paged import REFUSALS
from test_paged_gpu import _run_plan, _same_plan
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


@pytest.mark.parametrize("tokens", [2**31 - 1, 2**31 - (1 << 18) + 7])
def test_a_plan_of_nearly_2_to_the_31_rows(tn, tokens):
    """The rows' loop ends where another stride would pass 2^31: slots and positions to the last, and nothing ahead of
    them."""
    from torchnative_amd import _lib as L

    lib, guard = L.lib(), 1 << 18
    rows = tn.empty((2, guard + tokens), "int32", "hip")  # both outputs, each behind ints that no row is at
    at = [rows.data_ptr() + 4 * (i * (guard + tokens) + guard) for i in range(2)]
    L.check(lib.tn_memset(rows.data_ptr(), 0x55, rows.nbytes, None))
    up = lambda a: tn.tensor(np.asarray(a, np.int32), device="hip")  # noqa: E731
    width, pages, size = 20, 20, 256
    fresh, lens, table = up([3000, 5, 100]), up([10, 0, 20]), up(np.array([[7] + [-1] * (width - 1)] * 3))
    free, state, start, base = up(np.arange(pages)), up([pages, 0]), up([0] * 4), up([0] * 3)
    p = lambda t: t.data_ptr()  # noqa: E731
    print("tokens", tokens, flush=True)
    L.check(lib.tn_paged_plan(None, 3, p(fresh), p(lens), p(lens), p(table), width, size, p(free), pages, p(state),
                              p(state), tokens, p(start), p(base), at[0], at[1]))
    tn.synchronize()

    def ints(ptr, n):
        a = np.empty(n, np.int32)
        L.check(lib.tn_memcpy_d2h(a.ctypes.data, ptr, a.nbytes, None))
        return a

    want = P.plan(np.array([3000, 5, 100]), np.array([10, 0, 20]), np.array([[7] + [-1] * (width - 1)] * 3), size,
                  np.arange(pages), np.array([pages, 0]), 4000)
    for ptr, name, none in zip(at, ("slots", "pos"), (-1, 0)):
        assert np.array_equal(ints(ptr, 4000), want[name])
        for i in (4000, tokens // 2, tokens - (1 << 19)):
            assert (ints(ptr + 4 * i, 1 << 19) == none).all(), (name, i)
        assert (ints(ptr - 4 * guard, guard) == 0x55555555).all(), name


@pytest.mark.parametrize("lens, fresh, tokens, base, after, state", REFUSALS)
@pytest.mark.parametrize("behind", [0, 300, 2000])
def test_every_refusal_shows_in_the_state(tn, behind, lens, fresh, tokens, base, after, state):
    """behind: requests more, which add nothing (each workgroup size, and sums over several turns of it)."""
    n = len(lens) + behind
    lens, fresh = (np.array(x + [0] * behind, np.int32) for x in (lens, fresh))
    args = (fresh, lens, np.full((n, 3), 8, np.int32), 16, np.array([3, 1, 4, 0, 5, 2, -1, -1, -1], np.int32),
            np.array([6, 0], np.int32), tokens)
    got = _run_plan(tn, *args)
    _same_plan(got, P.plan(*args))
    assert (got["base"].tolist()[: len(base)], got["state"].tolist()) == (base, state)


@pytest.mark.parametrize("how", ["rows", "table", "pages"])
def test_rows_of_a_refused_request_and_its_tokens_given_again(tn, how):
    """A refused request's rows get the attention of its earlier tokens (NaN where it has fewer), the others theirs; the
    same tokens in a later step get their own."""
    w = Loop(tn, seed=3)
    first, second = {"rows": ([20, 0, 40, 9], [10, 0, 88, 1]), "table": ([20, 0, 120, 9], [1, 0, 30, 1]),
                     "pages": ([96, 96, 120, 9], [1, 0, 8, 70])}[how]
    refused = {"rows": 2, "table": 2, "pages": 3}[how]
    for fresh in ([f if i == j else 0 for j, f in enumerate(first)] for i in range(4)):
        for part in (min(80, max(fresh)), max(fresh) - min(80, max(fresh))):  # at most TOKENS rows a step
            if part:
                step = [part if f else 0 for f in fresh]
                w.inputs()
                w.table.step(step)
                w.dev.append(w.k, w.v, w.table.slots)
                w.check(step, *w.dev.attend(w.q, w.table, TOKENS, MOST), f"filling {step}")
    w.inputs()
    w.table.step(second)
    w.dev.append(w.k, w.v, w.table.slots)
    out, lse = w.dev.attend(w.q, w.table, TOKENS, MOST)
    ref = w.check(second, out, lse, how)
    base = w.o["base"]
    assert base[refused] == -1 and w.o["state"][1] > 0 and (base[:refused] >= 0).all()
    a, z = w.o["row_start"][refused:refused + 2]
    assert z > a
    tol, ltol = P.tolerance("float32", np.nan_to_num(ref[0]), ref[1], *(np.nan_to_num(x) for x in ref[2:]), MOST, D)
    out, lse = out.numpy(), lse.numpy()
    none = np.isneginf(ref[1][a:z])  # more rows than it has tokens
    assert np.array_equal(np.isneginf(lse[a:z]), none) and np.isnan(out[a:z][none]).all()
    assert none.any() == (z - a > w.o["lens"][refused])
    some = a + np.flatnonzero(~none.any(1))
    assert (np.abs(out[some] - ref[0][some]) <= tol[some]).all() and (np.abs(lse[some] - ref[1][some]) <= ltol[some]).all()
    if how == "rows":  # fits once it is not behind the others' rows
        again = [0, 0, 40, 0]
    elif how == "table":
        again = [0, 0, 8, 0]
    else:
        again = [-1, 0, 0, 70]
    w.inputs()
    w.table.step(again)
    w.dev.append(w.k, w.v, w.table.slots)
    w.check(again, *w.dev.attend(w.q, w.table, TOKENS, MOST), "again")
    assert (w.o["base"][[i for i, f in enumerate(again) if f > 0]] >= 0).all()


def test_a_captured_step_with_counts_of_the_callers(tn):
    """The graph copies the caller's counts at every replay; eager steps between have their own."""
    from torchnative_amd import _lib as L

    lib, s = L.lib(), tn.Stream()
    with s:
        w = Loop(tn, seed=5)
        t = w.table
        mine = tn.tensor(np.zeros(N, np.int32), device="hip")
        out, lse = tn.zeros((TOKENS, H * G, D)), tn.zeros((TOKENS, H * G))
        work = tn.empty((w.dev.work_floats(N, TOKENS, H * G, TOKENS, MOST) + 1,), "float32", "hip")
        L.check(lib.tn_stream_begin_capture(s.handle))
        t.step(mine)
        w.dev.append(w.k, w.v, t.slots)
        w.dev.attend(w.q, t, TOKENS, MOST, work=work, out=out, lse=lse)
        graph = ctypes.c_void_p()
        L.check(lib.tn_stream_end_capture(s.handle, ctypes.byref(graph)))
        for i, fresh in enumerate([[40, 3, 0, 0], [1, 1, 17, 0], [1, -1, 1, 50], [1, 30, 1, 1], [-1, 1, 1, 1], [7, 1, 1, 1]]):
            w.inputs()
            if i % 3 == 2:
                t.step(fresh)
                w.dev.append(w.k, w.v, t.slots)
                got = w.dev.attend(w.q, t, TOKENS, MOST)
            else:
                w.write(mine, np.asarray(fresh, np.int32))
                L.check(lib.tn_graph_launch(s.handle, graph))
                got = out, lse
            s.synchronize()
            w.check(fresh, *got, f"step {i}")
        L.check(lib.tn_graph_destroy(graph))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_two_streams_attend_one_cache_at_once(tn, dtype):
    """Eager calls without buffers of their own, interleaved on two streams: scratch is a stream's."""
    rng = np.random.default_rng(1)
    heads, dim, lens = 4, 128, [1500, 700]
    t, dev = tn.PageTable(2, 100, 16, 200, 2200), tn.Q4Cache(200, 16, heads, dim)
    t.step(lens)
    k, v = (tn.tensor(rng.standard_normal((2200, heads, dim)).astype(np.float32), dtype=dtype, device="hip") for _ in "kv")
    dev.append(k, v, t.slots)
    t.step([1, 1])
    dev.append(k, v, t.slots)
    qs = [tn.tensor(rng.standard_normal((2, 4 * heads, dim)).astype(np.float32), dtype=dtype, device="hip")
          for _ in range(6)]
    want = [[x.bits() for x in dev.attend(q, t, 1, 1600)] for q in qs]
    tn.synchronize()
    streams, got = (tn.Stream(), tn.Stream()), []
    for rnd in range(3):
        for i, q in enumerate(qs):
            with streams[i % 2]:
                got.append((i, dev.attend(q, t, 1, 1600)))
    tn.synchronize()
    for i, pair in got:
        assert all(np.array_equal(x.bits(), y) for x, y in zip(pair, want[i])), i
