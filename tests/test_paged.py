"""The paged 4-bit cache off the GPU: every refusal comes before a HIP call, empty calls touch no pointer, the oracle's
planes and blocks agree with the q4_0 codec's oracle, and the page bookkeeping holds its invariants."""

import ctypes

import numpy as np
import pytest

import oracle as O
from oracle import paged as P
from torchnative_amd import _lib


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _cache(pages=8, size=16, heads=2, dim=64, planes=(16, 16, 16, 16)):
    return _lib.Q4Cache(*planes, pages, size, heads, dim)


def _plan(L, n=1, width=4, size=16, pages=8, tokens=4, ptr=16, state=16):
    return L.tn_paged_plan(None, n, ptr, ptr, ptr, ptr, width, size, ptr, pages, state, state, tokens, ptr, ptr, ptr,
                           ptr)


def test_plan_refusals(L):
    for size in (0, 8, 24, 48, 512, -16):
        assert _plan(L, size=size) == _lib.TN_ENOTIMPL and f"page_size {size}" in _lib.last_error()
    assert _plan(L, n=4097) == _lib.TN_ENOTIMPL and "4097 requests" in _lib.last_error()
    for kw in ({"n": -1}, {"width": -1}, {"tokens": -1}, {"pages": -1}):
        assert _plan(L, **kw) == _lib.TN_EINVAL, kw
    for kw in ({"pages": 1 << 27}, {"width": 1 << 27}, {"tokens": 1 << 31}):
        assert _plan(L, **kw) == _lib.TN_EVALUE, kw
    assert _plan(L, ptr=None) == _lib.TN_EVALUE and "null pointer" in _lib.last_error()
    assert _plan(L, n=0, tokens=0, state=None) == _lib.TN_EVALUE


@pytest.mark.parametrize("kw, code, word", [
    ({"size": 24}, _lib.TN_ENOTIMPL, "page_size 24"),
    ({"dim": 80}, _lib.TN_ENOTIMPL, "head_dim 80"),
    ({"dim": 0}, _lib.TN_ENOTIMPL, "head_dim 0"),
    ({"dim": 288}, _lib.TN_ENOTIMPL, "head_dim 288"),
    ({"heads": 0}, _lib.TN_EINVAL, "bad cache sizes"),
    ({"pages": -1}, _lib.TN_EINVAL, "bad cache sizes"),
    ({"pages": 1 << 27}, _lib.TN_EVALUE, "2^31 slots"),
    ({"planes": (16, 16, None, 16)}, _lib.TN_EVALUE, "null cache plane"),
    ({"planes": (16, 16, 16, 8)}, _lib.TN_EVALUE, "16-byte aligned"),
])
def test_cache_refusals_at_every_entry(L, kw, code, word):
    c = ctypes.byref(_cache(**kw))
    nan = float("nan")
    for st in (L.tn_kv_append_q4_0(None, c, _lib.TN_F32, 16, 16, 1, 4096, 16),
               L.tn_kv_read_q4_0(None, c, 16, 1, _lib.TN_F32, 16, 16),
               L.tn_sdpa_paged_q4_0(None, c, _lib.TN_F32, 16, 4096, 1, 4 * max(1, kw.get("heads", 2)), 1, 16, 16, 16, 4,
                                    1, 16, nan, 16, 1 << 40, 16, 16)):
        assert st == code and word in _lib.last_error()
    for st in (L.tn_kv_append_q4_0(None, None, _lib.TN_F32, 16, 16, 1, 4096, 16),
               L.tn_kv_read_q4_0(None, None, 16, 1, _lib.TN_F32, 16, 16)):
        assert st == _lib.TN_EVALUE and "null cache" in _lib.last_error()


def test_row_refusals(L):
    c = ctypes.byref(_cache())
    for dt in (_lib.TN_F64, _lib.TN_BOOL, 99):
        assert L.tn_kv_append_q4_0(None, c, dt, 16, 16, 1, 128, 16) == _lib.TN_ENOTIMPL
        assert "float32, bfloat16 or float16" in _lib.last_error()
        assert L.tn_kv_read_q4_0(None, c, 16, 1, dt, 16, 16) == _lib.TN_ENOTIMPL
    assert L.tn_kv_append_q4_0(None, c, 0, 16, 16, -1, 128, 16) == _lib.TN_EINVAL
    assert L.tn_kv_append_q4_0(None, c, 0, 16, 16, 2, 127, 16) == _lib.TN_EINVAL and "row stride" in _lib.last_error()
    assert L.tn_kv_append_q4_0(None, c, 0, 16, 16, 2, 1 << 62, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q4_0(None, c, 0, 16, 16, 1 << 31, 128, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q4_0(None, c, 0, None, 16, 1, 128, 16) == _lib.TN_EVALUE
    assert L.tn_kv_read_q4_0(None, c, 16, 1, 0, None, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q4_0(None, c, 0, None, None, 0, 128, None) == _lib.TN_OK  # no rows: no pointer is touched
    assert L.tn_kv_read_q4_0(None, c, None, 0, 0, None, None) == _lib.TN_OK


def test_attention_refusals(L):
    c = ctypes.byref(_cache())

    def call(dtype=0, q=16, stride=256, tokens=2, Hq=4, n=1, starts=16, lens=16, table=16, width=4, rows=2, most=64,
             work=16, floats=1 << 40, out=16):
        return L.tn_sdpa_paged_q4_0(None, c, dtype, q, stride, tokens, Hq, n, starts, lens, table, width, rows, most,
                                    float("nan"), work, floats, out, None)

    assert call(dtype=_lib.TN_F64) == _lib.TN_ENOTIMPL and "float32, bfloat16 or float16" in _lib.last_error()
    assert call(Hq=3) == _lib.TN_ENOTIMPL and "do not divide" in _lib.last_error()
    for kw in ({"tokens": -1}, {"n": -1}, {"rows": -1}, {"most": -1}, {"Hq": -2}, {"width": -1}, {"most": 65},
               {"stride": 255}):
        assert call(**kw) == _lib.TN_EINVAL, kw
    for kw in ({"n": 65536}, {"tokens": 1 << 31}, {"tokens": 1 << 30}, {"Hq": 65536}, {"stride": 1 << 62}):
        assert call(**kw) == _lib.TN_EVALUE, kw
    for kw in ({"q": None}, {"out": None}, {"starts": None}, {"lens": None}, {"table": None}):
        assert call(**kw) == _lib.TN_EVALUE and "null pointer" in _lib.last_error(), kw
    assert call(work=8) == _lib.TN_EVALUE and "aligned" in _lib.last_error()
    need = L.tn_sdpa_paged_q4_0_work_floats(c, 1, 2, 4, 2, 64)
    assert need >= 0
    if need:
        assert call(floats=need - 1) == _lib.TN_EVALUE and f"needs {need}" in _lib.last_error()
        assert call(work=None) == _lib.TN_EVALUE
    for kw in ({"tokens": 0}, {"n": 0}, {"rows": 0}, {"Hq": 0}):  # nothing to compute: no pointer is touched
        assert call(**kw, q=None, out=None, starts=None, lens=None, table=None) == _lib.TN_OK, kw


def test_sizes_past_a_grid_are_refused(L):
    """A grid holds fewer than 2^32 threads in its first dimension and 2^16 workgroups in its second."""
    c = ctypes.byref(_cache())
    for m in ((1 << 28) + 1, (1 << 29) + 1, 1 << 30):
        assert L.tn_kv_append_q4_0(None, c, 0, 16, 16, m, 128, 16) == _lib.TN_EVALUE and "too large" in _lib.last_error()
        assert L.tn_kv_read_q4_0(None, c, 16, m, 0, 16, 16) == _lib.TN_EVALUE and "too large" in _lib.last_error()
    for heads in (4097, 8192):
        assert L.tn_kv_read_q4_0(None, ctypes.byref(_cache(heads=heads)), 16, 1, 0, 16, 16) == _lib.TN_EINVAL
    many = ctypes.byref(_cache(heads=4096, pages=1))
    for most in ((1 << 30) + 1, 1 << 31):
        args = (None, c, 0, 16, 256, 2, 4, 1, 16, 16, 16, 1 << 28, 2, most, float("nan"), 16, 1 << 60, 16, None)
        assert L.tn_sdpa_paged_q4_0(*args) == _lib.TN_EVALUE and "too large" in _lib.last_error()
    for n, rows in ((513, 2), (1024, 200), (65535, 1)):
        args = (None, many, 0, 16, 1 << 30, n, 4096, n, 16, 16, 16, 4, rows, 16, float("nan"), 16, 1 << 60, 16, None)
        assert L.tn_sdpa_paged_q4_0(*args) == _lib.TN_EVALUE and "too large" in _lib.last_error()


def test_work_never_shrinks_with_the_bounds(L):
    """A buffer made for a loop's largest step serves every smaller one: fewer requests, rows or tokens and shorter
    lengths never need more."""
    for dim in (64, 128):
        c = ctypes.byref(_cache(pages=1 << 16, heads=4, dim=dim))
        f = lambda n, T, rows, most: L.tn_sdpa_paged_q4_0_work_floats(c, n, T, 16, rows, most)  # noqa: E731
        for n, T, rows, most in ((16, 16, 1, 5000), (16, 700, 300, 5000), (300, 300, 1, 20000)):
            whole = f(n, T, rows, most)
            for less in ((1, 1, 1, most), (n // 2, T // 2, rows, most), (n, T, max(1, rows // 2), most),
                         (n, T, rows, most // 3), (1, T, rows, most)):
                assert f(*less) <= whole, (n, T, rows, most, less)


@pytest.mark.parametrize("D", [32, 96, 256])
def test_the_oracles_blocks_are_q4_0s(D):
    rng = np.random.default_rng(D)
    x = rng.standard_normal((40, D)).astype(np.float32)
    x[3] = 0
    x[4, :32] = [1.5, -1.5] * 16  # ties of size: the first decides the sign
    x[5] *= 1e-30
    code, d = P.blocks(x)
    blob = np.frombuffer(O.q4_0_quantize(x), np.uint8).reshape(-1, 18)
    assert np.array_equal(blob[:, :2].copy().view(np.float16).ravel().view(np.uint16), d.ravel().view(np.uint16))
    byte = code.reshape(-1, 32)
    assert np.array_equal(blob[:, 2:], byte[:, :16] | (byte[:, 16:] << 4))


def test_the_scale_saturates_and_nothing_cached_is_infinite():
    x = np.array([[3e38, -np.inf, 1e6, 7.0] + [0.0] * 28, [np.nan] * 32, [-65504.0] + [8188.0] * 31], np.float32)
    code, d = P.blocks(x)
    y = P.values(code, d)
    assert np.isfinite(y).all() and np.abs(y).max() == 65504
    assert y[2, 0] == -65504 and (np.abs(y[2, 1:] - 8188) <= 4094).all()


@pytest.mark.parametrize("seed", range(6))
def test_the_oracles_bookkeeping_keeps_every_page_once(seed):
    rng = np.random.default_rng(seed)
    n, S, width, pages = 9, 16, 6, 30
    lens, table = np.zeros(n, np.int32), np.full((n, width), -1, np.int32)
    free, state = rng.permutation(pages).astype(np.int32), np.array([pages, 0], np.int32)
    for _ in range(40):
        fresh = rng.integers(-1, 40, n).astype(np.int32)
        o = P.plan(fresh, lens, table, S, free, state, 120)
        assert (o["lens"] <= width * S).all()
        lens, table, free, state = o["lens"], o["table"], o["free"], o["state"]
        held = [table[r, : -(-lens[r] // S)] for r in range(n)]
        every = np.concatenate([free[: state[0]], *held])
        assert sorted(every) == list(range(pages))
        live = o["slots"][o["slots"] >= 0]
        assert len(set(live)) == len(live)


# lengths, fresh, tokens -> base, lens, state behind the step, of requests of up to three pages of 16 and six free ones
REFUSALS = [
    ([5, 5], [3, 4], 5, [5, -1], [8, 5], [6, 1]),           # rows past `tokens` that its last page would hold
    ([5, 5, 0], [3, 4, 0], 5, [5, -1, -1], [8, 5, 0], [6, 1]),  # and one behind it that adds nothing
    ([5, 40], [3, 20], 99, [5, -1], [8, 40], [6, 1]),       # a table row that is full
    ([0, 48], [1, 1], 99, [0, -1], [1, 48], [5, 1]),        # one that was full already
    ([16, 0, 0], [33, 48, 48], 99, [-1, 0, -1], [16, 48, 0], [3, 6]),
    ([0, 0, 0, 3], [48, 40, 2, 2], 99, [0, 0, -1, 3], [48, 40, 0, 5], [0, 1]),  # pages
    ([5, 5], [3, 0], 3, [5, 5], [8, 5], [6, 0]),
    ([5, 5], [-1, 3], 3, [0, 5], [0, 8], [7, 0]),
]


@pytest.mark.parametrize("lens, fresh, tokens, base, after, state", REFUSALS)
def test_every_refusal_shows_in_the_state(lens, fresh, tokens, base, after, state):
    n = len(lens)
    o = P.plan(np.array(fresh, np.int32), np.array(lens, np.int32), np.full((n, 3), 8, np.int32), 16,
               np.array([3, 1, 4, 0, 5, 2, -1, -1, -1], np.int32), np.array([6, 0], np.int32), tokens)
    assert (o["base"].tolist(), o["lens"].tolist(), o["state"].tolist()) == (base, after, state)


def _short_rows(rows, length, D, seed=0):
    """bf16 queries of the last rows of a request, its cache, and the oracle's arguments."""
    rng = np.random.default_rng(seed)
    c = P.Cache(-(-length // 16), 16, 1, D)
    c.append(*(rng.standard_normal((length, 1, D)).astype(np.float32) for _ in "kv"), np.arange(length))
    q = (rng.standard_normal((rows, 4, D)).astype(np.float32).view(np.uint32) & 0xffff0000).view(np.float32)
    return q.astype(np.float64), c, [0, rows], [length], np.arange(c.P)[None]


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_the_bound_of_rows_with_exact_keys_rejects_keys_rounded_to_f16(D):
    """The mistake is planted in the oracle: every key rounded. Rows of few keys show it, whose lse is nearly a score."""
    rows = length = 60
    args = _short_rows(rows, length, D)
    c = args[1]
    want = P.attend(*args)
    exact, stored = c.rows, {w: c.rows(w, np.arange(length)) for w in "kv"}
    c.rows = lambda w, slots: stored[w][slots].astype(np.float16).astype(np.float64) if w == "k" else exact(w, slots)
    got = P.attend(*args)
    keys = P.row_keys(*args[2:4], rows)
    assert keys.max() == length and (keys <= 1024).all()
    off = np.abs(got[1] - want[1])
    loose = P.tolerance("bfloat16", want[0], want[1], *want[2:], length, D)[1]
    tight = P.tolerance("bfloat16", want[0], want[1], *want[2:], length, D, rounded=keys > 1024, biased=False)[1]
    assert (off <= loose).all() and (off > tight).any()


def test_each_rows_keys():
    assert P.row_keys([0, 2, 2, 6], [5, 9, 2], 7).tolist() == [4, 5, 0, 0, 1, 2, 0]
