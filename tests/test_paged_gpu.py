"""The paged 4-bit cache on the GPU against oracle/paged.py: the bookkeeping and the written planes bit for bit, the
attention within bounds derived from its roundings (oracle.paged.tolerance)."""

import ctypes
import functools

import numpy as np
import pytest

from oracle import paged as P

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def tn():
    import torchnative_amd as tn

    print("device:", tn._hip_probe(), flush=True)
    return tn


def _up(tn, a, dtype=None):
    return tn.tensor(a, dtype=dtype, device="hip")


def _ints(tn, a):
    return tn.tensor(np.asarray(a, np.int32), device="hip")


# --- pages for requests ------------------------------------------------------------


def _run_plan(tn, fresh, lens, table, size, free, state, tokens, alias=False, stream=None):
    from torchnative_amd import _lib as L

    n = len(fresh)
    t = {k: _ints(tn, v) for k, v in (("fresh", fresh), ("lens", lens), ("table", table), ("free", free),
                                      ("state", state))}
    o = {"lens": t["lens"] if alias else _ints(tn, [-7] * n), "state": t["state"] if alias else _ints(tn, [-7, -7]),
         "row_start": _ints(tn, [-7] * (n + 1)), "base": _ints(tn, [-7] * n), "slots": _ints(tn, [-7] * tokens),
         "pos": _ints(tn, [-7] * tokens), "table": t["table"], "free": t["free"]}
    p = lambda x: x.data_ptr()  # noqa: E731
    L.check(L.lib().tn_paged_plan(stream, n, p(t["fresh"]), p(t["lens"]), p(o["lens"]), p(t["table"]), table.shape[1],
                                  size, p(t["free"]), len(free), p(t["state"]), p(o["state"]), tokens,
                                  p(o["row_start"]), p(o["base"]), p(o["slots"]), p(o["pos"])))
    tn.synchronize()
    return {k: v.numpy().reshape(np.shape(table) if k == "table" else -1) for k, v in o.items()}


def _same_plan(got, want, note=""):
    for k in want:
        assert np.array_equal(got[k], want[k]), f"{note} {k}: {got[k].ravel()[:20]} {np.ravel(want[k])[:20]}"


@pytest.mark.parametrize("n, size, width, pages, tokens, most", [
    (1, 16, 4, 3, 5, 6), (7, 16, 6, 20, 90, 40), (64, 32, 9, 300, 700, 30), (65, 64, 3, 100, 4096, 150),
    (1000, 16, 12, 6000, 9000, 20), (1025, 16, 40, 9000, 70000, 90), (4096, 256, 2, 5000, 4097, 3),
    (3, 128, 300, 900, 100001, 38400), (5, 16, 0, 8, 10, 3), (4, 16, 6, 0, 10, 3), (6, 16, 5, 40, 0, 3),
])
def test_plan_equals_the_sequential_bookkeeping(tn, n, size, width, pages, tokens, most):
    rng = np.random.default_rng(n + tokens)
    lens, table = np.zeros(n, np.int32), np.full((n, width), -1, np.int32)
    free, state = rng.permutation(pages).astype(np.int32), np.array([pages, 0], np.int32)
    for step in range(6):
        fresh = rng.integers(-(most // 3) - 1, most + 1, n).astype(np.int32)
        want = P.plan(fresh, lens, table, size, free, state, tokens)
        got = _run_plan(tn, fresh, lens, table, size, free, state, tokens, alias=step % 2 == 1)
        _same_plan(got, want, f"step {step}")
        lens, table, free, state = want["lens"], want["table"], want["free"], want["state"]


def test_plan_with_numbers_out_of_range(tn):
    """Lengths, counts and pages past their ranges are cut, and no slot outside the pool comes out."""
    table = np.array([[0, 99], [-5, 1], [2, 3]], np.int32)
    free = np.array([4, -9, 77, 5], np.int32)
    for state in ([9, 0], [-3, 0], [4, 0]):
        for lens in ([-4, 5, 1000], [32, 16, 17], [2**31 - 1, -2**31, 0]):
            for fresh in ([1, 2**31 - 1, 1], [20, -2**31, -1], [2**31 - 1] * 3):
                lens_, fresh_ = np.array(lens, np.int32), np.array(fresh, np.int32)
                want = P.plan(fresh_, lens_, table, 16, free, np.array(state, np.int32), 40)
                got = _run_plan(tn, fresh_, lens_, table, 16, free, np.array(state, np.int32), 40)
                _same_plan(got, want, f"{state} {lens} {fresh}")
                assert (got["slots"] < 64).all() and (got["slots"] >= -1).all()


# --- rows into the cache and back ------------------------------------------------------


def _device_cache(tn, c, fill=0):
    d = tn.Q4Cache(c.P, c.S, c.H, c.D)
    for t in (d.k_codes, d.k_scales, d.v_codes, d.v_scales):
        from torchnative_amd import _lib as L

        L.check(L.lib().tn_memset(t.data_ptr(), fill, t.nbytes, None))
    return d


def _planes(d):
    return [t.numpy().ravel().view(np.uint8) for t in (d.k_codes, d.k_scales, d.v_codes, d.v_scales)]


def _bytes(c):
    return [a.view(np.uint8) for a in c.planes()]


def _fill(tn, c, fill=0):
    """A device cache holding the oracle's planes."""
    d = tn.Q4Cache(c.P, c.S, c.H, c.D)
    from torchnative_amd import _lib as L

    for t, a in zip((d.k_codes, d.k_scales, d.v_codes, d.v_scales), c.planes()):
        a = np.ascontiguousarray(a)
        L.check(L.lib().tn_memcpy_h2d(t.data_ptr(), a.ctypes.data, a.nbytes, None))
    return d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, D, S, m", [(1, 32, 16, 1), (3, 64, 16, 50), (2, 96, 32, 33), (8, 128, 64, 200),
                                        (1, 160, 128, 17), (2, 192, 16, 9), (3, 224, 32, 31), (2, 256, 256, 300)])
def test_append_writes_the_planes_and_read_gives_them_back(tn, dtype, H, D, S, m):
    rng = np.random.default_rng(D + m)
    Pg = -(-m // S) + 2
    c = P.Cache(Pg, S, H, D)
    dev = _fill(tn, c)
    for order in ("ordered", "shuffled"):
        x = [rng.standard_normal((m, H, D)).astype(np.float32) * np.float32(10.0 ** rng.integers(-3, 3)) for _ in "kv"]
        x[0][0, 0, :32] = 0
        x[1][-1, -1, -32:] = np.tile([2.5, -2.5], 16)
        k, v = (_up(tn, a, dtype) for a in x)
        if order == "ordered":  # positions in order, from the middle of a page on
            slots = (np.arange(m) + S // 2 + 3).astype(np.int32) % (Pg * S)
        else:
            slots = rng.permutation(Pg * S)[:m].astype(np.int32)
        slots[m // 2] = [-1, Pg * S][m % 2]  # no row of the cache
        dev.append(k, v, _ints(tn, slots))
        c.append(k.numpy().astype(np.float32), v.numpy().astype(np.float32), slots)
        tn.synchronize()
        for name, got, want in zip(("kc", "kd", "vc", "vd"), _planes(dev), _bytes(c)):
            assert np.array_equal(got, want), f"{order} {name}: {np.flatnonzero(got != want)[:8]}"
        live = (slots >= 0) & (slots < Pg * S)
        for out in DTYPES:
            got = [t.numpy().astype(np.float64) for t in dev.read(_ints(tn, slots), out)]
            for w, y in zip("kv", got):
                want = _up(tn, c.rows(w, np.where(live, slots, 0)).astype(np.float32), out).numpy().astype(np.float64)
                assert np.array_equal(y[live], want[live]) and np.isnan(y[~live]).all()


def test_append_of_large_infinite_and_nan_values_saturates(tn):
    x = np.zeros((3, 1, 32), np.float32)
    x[0, 0, :4] = [3e38, -np.inf, 1e6, 7]
    x[1] = np.nan
    x[2, 0] = np.linspace(-70000, 60000, 32)
    c = P.Cache(1, 16, 1, 32)
    dev = _fill(tn, c)
    dev.append(_up(tn, x), _up(tn, x[::-1].copy()), _ints(tn, [0, 1, 2]))
    c.append(x, x[::-1], [0, 1, 2])
    for got, want in zip(_planes(dev), _bytes(c)):
        assert np.array_equal(got, want)
    assert all(np.isfinite(t.numpy()).all() for t in dev.read(_ints(tn, [0, 1, 2])))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_large_read_equals_its_pieces(tn, dtype):
    """Past 32 MB the output goes past the caches; the same values as a few rows at a time, NaN rows among them."""
    rng = np.random.default_rng(2)
    H, D, S, m = 8, 128, 64, 9001
    dev = tn.Q4Cache(-(-m // S), S, H, D)
    k = _up(tn, rng.standard_normal((m, H, D)).astype(np.float32), dtype)
    slots = rng.permutation(dev.pages)[np.arange(m) // S] * S + np.arange(m) % S
    dev.append(k, k, _ints(tn, slots))
    slots[77] = -1
    whole = [t.bits() for t in dev.read(_ints(tn, slots), dtype)]
    for a in range(0, m, 3001):
        for x, y in zip(whole, dev.read(_ints(tn, slots[a:a + 3001]), dtype)):
            assert x[a:a + 3001].tobytes() == y.bits().tobytes()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [31, 32, 33])
@pytest.mark.parametrize("many", [False, True])
def test_rows_around_the_kernels_limit(tn, many, dtype, rows):
    c = Case(tn, dtype, 2, 4, 64, 16, [rows, 32, 33], [600, 40, 90])
    c.check(c.run(tn, many=many))


def test_append_equals_the_linears_writer(tn):
    """The same blocks as tn_q4_0_quantize gives a weight of the same rows."""
    rng = np.random.default_rng(0)
    m, H, D = 24, 2, 128
    k, v = (rng.standard_normal((m, H, D)).astype(np.float32) for _ in range(2))
    dev = tn.Q4Cache(2, 16, H, D)
    dev.append(_up(tn, k), _up(tn, v), _ints(tn, np.arange(m)))
    for x, y in zip((k, v), dev.read(_ints(tn, np.arange(m)))):
        w = tn._dequantize(tn._quantize(_up(tn, x.reshape(m, -1)), "q4_0")).numpy()
        assert np.array_equal(y.numpy().reshape(m, -1), w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_parts_of_stacked_rows_at_any_alignment(tn, dtype):
    from torchnative_amd import _lib as L

    rng = np.random.default_rng(4)
    m, H, D, lead = 21, 2, 64, 3
    wide = 4 * H * D + 5  # q|k|v rows with an odd pitch
    flat = rng.standard_normal(lead + m * wide).astype(np.float32)
    x = _up(tn, flat, dtype)
    c = P.Cache(3, 16, H, D)
    dev = _fill(tn, c)
    slots = np.arange(5, 5 + m).astype(np.int32)
    size = x.element_size
    ko, vo = lead + 2 * H * D, lead + 3 * H * D
    L.check(L.lib().tn_kv_append_q4_0(None, ctypes.byref(dev._c), {"float32": 0, "bfloat16": 1, "float16": 2}[dtype],
                                      x.data_ptr() + ko * size, x.data_ptr() + vo * size, m, wide,
                                      _ints(tn, slots).data_ptr()))
    tn.synchronize()
    h = x.numpy().astype(np.float32)
    rows = lambda o: np.stack([h[o + t * wide: o + t * wide + H * D] for t in range(m)]).reshape(m, H, D)  # noqa: E731
    c.append(rows(ko), rows(vo), slots)
    for got, want in zip(_planes(dev), _bytes(c)):
        assert np.array_equal(got, want)


# --- attention --------------------------------------------------------------------------


class Case:
    """Requests with rows[r] rows and lens[r] cached tokens, their pages at random, everything outside of a request's
    tokens filled with bytes of 255 (scales that are NaN)."""

    def __init__(self, tn, dtype, H, G, D, S, rows, lens, seed=0, extra=0, spread=1.0):
        rng = np.random.default_rng(seed)
        self.dtype, self.D, self.S, self.Hq = dtype, D, S, H * G
        self.rows, self.lens = rows, lens
        held = [-(-x // S) for x in lens]
        width = max(held + [1]) + 1
        pages = rng.permutation(sum(held) + 3).astype(np.int32)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for r, h in enumerate(held):
            self.table[r, :h] = pages[at:at + h]
            at += h
        c = P.Cache(len(pages), S, H, D)
        for w in "kv":
            c.code[w][:], c.d[w][:] = 15, np.frombuffer(b"\xff\xff", np.float16)[0]
        for r, x in enumerate(lens):
            t = np.arange(x)
            slots = self.table[r, t // S] * S + t % S if x else np.zeros(0, np.int64)
            kv = [rng.standard_normal((x, H, D)).astype(np.float32) * np.float32(spread) for _ in "kv"]
            for w, y in zip("kv", kv):
                if x:
                    c.code[w][slots], c.d[w][slots] = P.blocks(y)
        self.cache = c
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        T = int(self.row_start[-1]) + extra
        self.q = _up(tn, rng.standard_normal((T, self.Hq, D)).astype(np.float32), dtype)
        self.max_rows, self.max_len = max(rows + [0]), max(lens + [0])

    def run(self, tn, dev=None, stream=None, scale=None, fill=7.5, lse=True, table=None, max_len=None, max_rows=None,
            bits=False, many=False):
        """many: the bound of a length is so loose that the call is one of many products, k_paged_many's."""
        from torchnative_amd import _lib as L

        dev = dev or _fill(tn, self.cache)
        T = self.q.shape[0]
        out = _up(tn, np.full(self.q.shape, fill, np.float32), self.dtype)
        ls = _up(tn, np.full((T, self.Hq), fill, np.float32))
        table = self.table if table is None else table
        if many:
            short = max(0, (1 << 34) // (T * self.Hq * self.D * self.S) + 1 - table.shape[1])
            table = np.pad(table, ((0, 0), (0, short)), constant_values=-1)
            max_len = table.shape[1] * self.S
        t = [_ints(tn, a) for a in (self.row_start, self.lens, table)]
        most, rows = max_len or self.max_len, max_rows or self.max_rows
        n = len(self.lens)
        floats = dev.work_floats(n, T, self.Hq, rows, most)
        work = _up(tn, np.full(floats + 1, np.nan, np.float32))
        print(f"case {self.dtype} heads {self.Hq}/{self.cache.H} D {self.D} S {self.S} rows {self.rows} lens "
              f"{self.lens} work {floats}", flush=True)
        L.check(L.lib().tn_sdpa_paged_q4_0(
            stream, ctypes.byref(dev._c), {"float32": 0, "bfloat16": 1, "float16": 2}[self.dtype], self.q.data_ptr(),
            self.Hq * self.D, T, self.Hq, n, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), table.shape[1],
            rows, most, float("nan") if scale is None else scale, work.data_ptr(), floats, out.data_ptr(),
            ls.data_ptr() if lse else None))
        tn.synchronize()
        if bits:
            return out.bits(), ls.bits()
        return out.numpy().astype(np.float64), ls.numpy().astype(np.float64)

    def check(self, got, scale=None, table=None, fill=7.5):
        out, lse = got
        ref = P.attend(self.q.numpy().astype(np.float64), self.cache, self.row_start, self.lens,
                       self.table if table is None else table, scale)
        ro, rl = ref[0], ref[1]
        keys = max(self.max_len, 1)
        with np.errstate(invalid="ignore"):
            tol, ltol = P.tolerance(self.dtype, np.nan_to_num(ro), rl, *(np.nan_to_num(x) for x in ref[2:]), keys,
                                    self.D)
        own = np.zeros(len(out), bool)
        own[: self.row_start[-1]] = True
        assert (out[~own] == fill).all() and (lse[~own] == fill).all(), "rows behind the last request were written"
        dead = np.isnan(ro)
        assert np.array_equal(np.isnan(out[own]), dead[own])
        assert np.array_equal(np.isnan(lse[own]), np.isnan(rl[own]))
        fin = np.isfinite(rl)
        assert np.array_equal(lse[own & ~np.isnan(rl).any(1)] == -np.inf, rl[own & ~np.isnan(rl).any(1)] == -np.inf)
        with np.errstate(invalid="ignore"):
            worst = np.max(np.where(own[:, None, None] & ~dead, np.abs(out - ro) / tol, 0), initial=0)
            lworst = np.max(np.where(own[:, None] & fin, np.abs(lse - rl) / ltol, 0), initial=0)
        print(f"  worst {worst:.3f} of the bound, lse {lworst:.3f}", flush=True)
        assert worst <= 1 and lworst <= 1, (worst, lworst)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(3, 3, 64, 16), (2, 4, 128, 16), (1, 1, 32, 32), (1, 7, 96, 64), (2, 8, 256, 128),
                                        (1, 2, 160, 16), (1, 3, 192, 256), (1, 5, 224, 32), (1, 20, 64, 16),
                                        (1, 16, 128, 32)])
def test_single_tokens(tn, dtype, H, G, D, S):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 127, 200]
    c = Case(tn, dtype, H, G, D, S, [1] * len(lens), lens, seed=D, extra=2)
    c.check(c.run(tn))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D, G, lens", [(64, 3, [3000]), (128, 4, [1, 2500, 700]), (96, 1, [1999, 4])])
def test_single_tokens_over_long_contexts(tn, dtype, D, G, lens):
    c = Case(tn, dtype, 2, G, D, 16, [1] * len(lens), lens, seed=D)
    c.check(c.run(tn))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(3, 3, 64, 16), (2, 4, 128, 64), (1, 6, 96, 16), (1, 1, 256, 32), (1, 2, 32, 16),
                                        (1, 2, 160, 16), (1, 1, 192, 32), (1, 1, 224, 16)])
@pytest.mark.parametrize("rows, lens", [
    ([130], [130]), ([3, 0, 70, 1], [90, 40, 70, 200]), ([2, 5, 4], [300, 5, 65]), ([33, 257], [33, 300]),
])
@pytest.mark.parametrize("many", [False, True])
def test_chunks_and_whole_prompts(tn, many, dtype, H, G, D, S, rows, lens):
    c = Case(tn, dtype, H, G, D, S, rows, lens, seed=D + len(rows), extra=3)
    c.check(c.run(tn, many=many))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(2, 3, 64, 16), (1, 4, 128, 32), (1, 2, 96, 16), (1, 1, 256, 64), (1, 2, 32, 16)])
@pytest.mark.parametrize("rows, lens", [([90], [2100]), ([200, 1, 0, 70, 3], [1500, 900, 40, 70, 1033])])
@pytest.mark.parametrize("many", [False, True])
def test_chunks_behind_long_contexts(tn, many, dtype, H, G, D, S, rows, lens):
    """Keys split over workgroups, with rows whose part of the keys is empty."""
    c = Case(tn, dtype, H, G, D, S, rows, lens, seed=D + len(rows), extra=2)
    c.check(c.run(tn, many=many))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("rows", [[250, 1, 600, 0, 700, 513], [150, 1, 300, 0, 350, 199]])
def test_many_rows_of_many_heads(tn, dtype, D, rows):
    """More than 65536 folded rows: the kernel of 256 rows a workgroup, with a request of few rows among the others;
    and a little fewer, in workgroups of 128 that take whole rows' keys."""
    c = Case(tn, dtype, 8, 8, D, 32, rows, [260, 500, 610, 3, 690, 513], seed=D)
    c.check(c.run(tn, many=True))


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("H, G", [(8, 8), (2, 2)])
def test_rows_of_many_keys(tn, D, H, G):
    """bfloat16 rows from where one part of a key does: some workgroups of a request on either side."""
    rows = [700, 600, 800] if H == 8 else [300, 5, 70]
    c = Case(tn, "bfloat16", H, G, D, 32, rows, [1500, 1623, 800] if H == 8 else [1200, 1500, 3001], seed=D)
    c.check(c.run(tn, many=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("many", [False, True])
def test_rows_without_keys_and_empty_requests(tn, many, dtype):
    """More rows than tokens: the first attend nothing. Requests of no rows, of no tokens, and of neither."""
    c = Case(tn, dtype, 2, 2, 64, 16, [5, 1, 0, 0, 40, 20], [2, 0, 33, 0, 17, 0], extra=1)
    got = c.run(tn, many=many)
    c.check(got)
    assert np.isnan(got[0][:3]).all() and (got[1][:3] == -np.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[1, 1, 2], [40, 3, 200], [300]])
@pytest.mark.parametrize("many", [False, True])
def test_rows_past_the_calls_are_cut(tn, many, dtype, rows):
    """row_start from below zero to past the last row is as if it ran from zero to it."""
    c = Case(tn, dtype, 2, 2, 64, 16, rows, [x + 70 for x in rows])
    c.row_start[0], c.row_start[-1] = -5, c.row_start[-1] + 1000
    got = c.run(tn, many=many)
    c.row_start[0], c.row_start[-1] = 0, c.q.shape[0]
    c.check(got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("many", [False, True])
def test_a_page_outside_the_cache_makes_its_rows_nan(tn, many, dtype, rows):
    c = Case(tn, dtype, 1, 2, 64, 16, [rows, rows, rows], [100, 100, 100])
    for bad in (-1, c.cache.P, 2**31 - 1, -2**31):
        table = c.table.copy()
        table[1, 5] = bad  # tokens 80 .. 95
        got = c.run(tn, table=table, many=many)
        c.check(got, table=table)
        first = np.isnan(got[0]).all((1, 2))
        assert not first[:rows].any() and not first[2 * rows:].any() and first[2 * rows - 1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 75])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 8.0])
@pytest.mark.parametrize("many", [False, True])
def test_scales_of_any_sign_and_peaked_rows(tn, many, dtype, rows, scale):
    c = Case(tn, dtype, 2, 3, 64, 16, [rows, rows], [150, 75], seed=5)
    c.check(c.run(tn, scale=scale, many=many), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 75])
@pytest.mark.parametrize("spread", [1e-4, 300.0, 10000.0])
@pytest.mark.parametrize("many", [False, True])
def test_small_and_large_values(tn, many, dtype, rows, spread):
    """Scores of one sign past thousands, values from f16's subnormal scales to near its largest."""
    c = Case(tn, dtype, 1, 4, 128, 32, [rows], [180], seed=6, spread=spread)
    scale = 0.1 / spread if spread > 1 else None
    c.check(c.run(tn, scale=scale, many=many), scale=scale)


@pytest.mark.parametrize("many", [False, True])
def test_large_queries_of_each_type(tn, many):
    """Queries of 1e30 (f32, bf16) and 6e4 (f16) with a scale that brings the scores back; 1e-30 likewise."""
    for dtype, mul in (("float32", 1e30), ("bfloat16", 1e30), ("float16", 6e4), ("float32", 1e-30),
                       ("bfloat16", 1e-30)):
        for rows in (1, 70):
            c = Case(tn, dtype, 1, 2, 64, 16, [rows], [90], seed=8)
            x = np.clip(c.q.numpy().astype(np.float32), -1, 1) * np.float32(mul)
            c.q = _up(tn, x, dtype)
            c.check(c.run(tn, scale=0.125 / mul, many=many), scale=0.125 / mul)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_lse_and_a_shared_prefix(tn, dtype):
    c = Case(tn, dtype, 2, 2, 64, 16, [1, 1, 20], [64, 80, 90])
    c.table[1, :4] = c.table[0, :4]  # the second and third request share the first one's pages
    c.table[2, :4] = c.table[0, :4]
    got = c.run(tn)
    c.check(got)
    out, lse = c.run(tn, lse=False)
    assert np.array_equal(out, got[0]) and (lse == 7.5).all()


@pytest.mark.parametrize("rows", [[1, 1, 1], [90, 1, 4]])
@pytest.mark.parametrize("many", [False, True])
def test_the_same_bits_every_time_and_whatever_the_bounds_hold(tn, many, rows):
    c = Case(tn, "bfloat16", 2, 4, 128, 16, rows, [900, 1300, 40])
    first = c.run(tn, bits=True, many=many)
    for _ in range(3):
        again = c.run(tn, bits=True, many=many)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("rows", [[1, 1], [64, 3]])
def test_loose_bounds_give_the_result_within_the_bound(tn, rows):
    c = Case(tn, "float16", 1, 4, 64, 16, rows, [100, 130])
    c.check(c.run(tn, max_len=(c.table.shape[1]) * 16, max_rows=500))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 66])
def test_query_rows_inside_stacked_rows(tn, dtype, rows):
    from torchnative_amd import _lib as L

    c = Case(tn, dtype, 2, 2, 96, 16, [rows, rows], [70, 130])
    want = c.run(tn, bits=True)
    T, Hq, D = c.q.shape
    wide, lead = Hq * D + 7, 5
    x = np.full(lead + T * wide, np.nan, np.float32)
    for t in range(T):
        x[lead + t * wide: lead + t * wide + Hq * D] = c.q.numpy()[t].ravel()
    x = _up(tn, x, dtype)
    dev = _fill(tn, c.cache)
    out, lse = tn.empty(c.q.shape, dtype, "hip"), tn.empty((T, Hq), "float32", "hip")
    t = [_ints(tn, a) for a in (c.row_start, c.lens, c.table)]
    floats = dev.work_floats(2, T, Hq, c.max_rows, c.max_len)
    work = tn.empty((floats + 1,), "float32", "hip")
    L.check(L.lib().tn_sdpa_paged_q4_0(
        None, ctypes.byref(dev._c), {"float32": 0, "bfloat16": 1, "float16": 2}[dtype],
        x.data_ptr() + lead * x.element_size, wide, T, Hq, 2, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(),
        c.table.shape[1], c.max_rows, c.max_len, float("nan"), work.data_ptr(), floats, out.data_ptr(),
        lse.data_ptr()))
    tn.synchronize()
    assert np.array_equal(out.bits(), want[0]) and np.array_equal(lse.bits(), want[1])


# --- a run of them together ------------------------------------------------------------------


def _loop(tn, steps, stream, capture, seed=0):
    """A serving loop of prompts and single tokens, ended requests and new ones: each step plans, appends and attends.
    Returns every step's (lens, out, lse) and the oracle's."""
    rng = np.random.default_rng(seed)
    n, H, G, D, S, width, pages, tokens = 4, 2, 3, 64, 16, 8, 24, 96
    table = tn.PageTable(n, width, S, pages, tokens)
    dev = tn.Q4Cache(pages, S, H, D)
    k, v = (tn.zeros((tokens, H, D)) for _ in range(2))
    q = tn.zeros((tokens, H * G, D))
    out, lse = tn.zeros((tokens, H * G, D)), tn.zeros((tokens, H * G))
    most = width * S
    work = tn.empty((dev.work_floats(n, tokens, H * G, tokens, most) + 1,), "float32", "hip")
    from torchnative_amd import _lib as L

    lib = L.lib()

    def write(t, a):
        a = np.ascontiguousarray(a)
        L.check(lib.tn_memcpy_h2d(t.data_ptr(), a.ctypes.data, a.nbytes, stream.handle))

    def step():
        table.step()
        dev.append(k, v, table.slots)
        dev.attend(q, table, tokens, most, work=work, out=out, lse=lse)

    oc = P.Cache(pages, S, H, D)
    o = {"lens": np.zeros(n, np.int32), "table": np.full((n, width), -1, np.int32),
         "free": np.arange(pages, dtype=np.int32)[::-1].copy(), "state": np.array([pages, 0], np.int32)}
    graph = None
    with stream:
        if capture:
            L.check(lib.tn_stream_begin_capture(stream.handle))
            step()
            graph = ctypes.c_void_p()
            L.check(lib.tn_stream_end_capture(stream.handle, ctypes.byref(graph)))
        for i, fresh in enumerate(steps):
            fresh = np.asarray(fresh, np.int32)
            kv = [rng.standard_normal((tokens, H, D)).astype(np.float32) for _ in "kv"]
            qq = rng.standard_normal((tokens, H * G, D)).astype(np.float32)
            for t, a in zip((table.fresh, k, v, q), (fresh, *kv, qq)):
                write(t, a)
            if capture:
                L.check(lib.tn_graph_launch(stream.handle, graph))
            else:
                step()
            stream.synchronize()
            o = P.plan(fresh, o["lens"], o["table"], S, o["free"], o["state"], tokens)
            oc.append(*kv, o["slots"])
            assert np.array_equal(table.lens.numpy(), o["lens"]) and np.array_equal(table.state.numpy(), o["state"])
            assert np.array_equal(table.slots.numpy(), o["slots"]) and np.array_equal(table.pos.numpy(), o["pos"])
            ref = P.attend(qq.astype(np.float64), oc, o["row_start"], o["lens"], o["table"])
            tol, ltol = P.tolerance("float32", np.nan_to_num(ref[0]), ref[1], *(np.nan_to_num(x) for x in ref[2:]), most, D)
            live = o["slots"] >= 0
            assert (np.abs(out.numpy()[live] - ref[0][live]) <= tol[live]).all(), f"step {i}"
            assert (np.abs(lse.numpy()[live] - ref[1][live]) <= ltol[live]).all(), f"step {i}"
            yield out.bits(), lse.bits()
    if graph is not None:
        L.check(lib.tn_graph_destroy(graph))


STEPS = [[40, 3, 0, 0], [1, 1, 17, 0], [1, 1, 1, 50], [1, -1, 1, 1], [1, 30, 1, 1], [-1, 1, 1, 1], [60, 1, -1, 1],
         [1, 1, 5, 1], [90, 90, 1, 1], [1, 1, 1, 1]]


def test_a_serving_loop_eager_and_captured(tn):
    eager = list(_loop(tn, STEPS, tn.Stream(), False))
    graph = list(_loop(tn, STEPS, tn.Stream(), True))
    for i, (a, b) in enumerate(zip(eager, graph)):
        assert all(x.tobytes() == y.tobytes() for x, y in zip(a, b)), f"step {i}"


def test_two_graphs_replayed_at_once_on_two_streams(tn):
    """Each with its own work buffer, replayed side by side several times with eager work of the same streams between."""
    from torchnative_amd import _lib as L

    lib = L.lib()
    runs = []
    for seed, lens in ((1, [2000, 700]), (2, [1500, 90])):
        c = Case(tn, "bfloat16", 2, 4, 128, 16, [1, 1], lens, seed=seed)
        want = c.run(tn, bits=True)
        dev, T = _fill(tn, c.cache), 2
        t = [_ints(tn, a) for a in (c.row_start, c.lens, c.table)]
        out, lse = tn.zeros(c.q.shape, "bfloat16"), tn.zeros((T, c.Hq))
        floats = dev.work_floats(2, T, c.Hq, 1, c.max_len)
        work = tn.empty((floats + 1,), "float32", "hip")
        s = tn.Stream()
        call = functools.partial(
            lib.tn_sdpa_paged_q4_0, s.handle, ctypes.byref(dev._c), 1, c.q.data_ptr(), c.Hq * c.D, T, c.Hq, 2,
            t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), c.table.shape[1], 1, c.max_len, float("nan"),
            work.data_ptr(), floats, out.data_ptr(), lse.data_ptr())
        tn.synchronize()
        L.check(lib.tn_stream_begin_capture(s.handle))
        L.check(call())
        graph = ctypes.c_void_p()
        L.check(lib.tn_stream_end_capture(s.handle, ctypes.byref(graph)))
        runs.append((s, graph, out, lse, want, call, (c, dev, t, work)))
    for rnd in range(4):
        for _, _, out, lse, *_ in runs:
            out.zero_(), lse.zero_()
        tn.synchronize()
        for _ in range(5):
            for s, graph, *_ in runs:
                L.check(lib.tn_graph_launch(s.handle, graph))
        if rnd % 2:
            for *_, call, _ in runs:
                L.check(call())
        for s, *_ in runs:
            s.synchronize()
        for _, _, out, lse, want, *_ in runs:
            assert np.array_equal(out.bits(), want[0]) and np.array_equal(lse.bits(), want[1]), rnd
    for _, graph, *_ in runs:
        L.check(lib.tn_graph_destroy(graph))


def test_a_cache_past_four_gigabytes(tn):
    """Pages whose bytes lie behind 2^32: the same result as from the first pages."""
    H, D, S = 8, 256, 256
    pages = (1 << 32) // (H * S * D // 2) + 40
    small = Case(tn, "bfloat16", H, 1, D, S, [1, 9], [700, 300], seed=3)
    far = tn.Q4Cache(pages, S, H, D)
    near = _fill(tn, small.cache)
    from torchnative_amd import _lib as L

    shift = pages - small.cache.P
    for a, b in zip((near.k_codes, near.k_scales, near.v_codes, near.v_scales),
                    (far.k_codes, far.k_scales, far.v_codes, far.v_scales)):
        L.check(L.lib().tn_memcpy_d2d(b.data_ptr() + b.nbytes - a.nbytes, a.data_ptr(), a.nbytes, None))
    want = small.run(tn, dev=near, bits=True)
    table = np.where(small.table >= 0, small.table + shift, -1)
    got = small.run(tn, dev=far, table=table, bits=True)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))
    # and rows written there
    rng = np.random.default_rng(1)
    k, v = (_up(tn, rng.standard_normal((4, H, D)).astype(np.float32)) for _ in range(2))
    at = np.array([pages * S - 1, pages * S - 9, (pages - 1) * S, shift * S + 3], np.int32)
    far.append(k, v, _ints(tn, at))
    near.append(k, v, _ints(tn, at - shift * S))
    for a, b in zip(far.read(_ints(tn, at)), near.read(_ints(tn, at - shift * S))):
        assert np.array_equal(a.numpy(), b.numpy()) and np.isfinite(a.numpy()).all()
