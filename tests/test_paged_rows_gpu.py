"""Rows of the paged attention at the edges of a call: ahead of the first request's, past the bounds on rows and
lengths, queries that are not finite."""

import numpy as np
import pytest

from oracle import paged as P
from test_paged_gpu import DTYPES, Case, _up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tn():
    import torchnative_amd as tn

    return tn


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, lens", [([1, 1], [70, 900]), ([90], [2100]), ([200, 1, 0, 70, 3], [1500, 900, 40, 70, 1033])])
@pytest.mark.parametrize("lead", [1, 37])
@pytest.mark.parametrize("many", [False, True])
def test_rows_ahead_of_the_first_request_are_left_as_they_were(tn, many, lead, dtype, rows, lens):
    """A call over the later requests of a step: row_start[0] is where their rows begin. Few and many rows, keys split
    and not."""
    c = Case(tn, dtype, 2, 2, 64, 16, rows, lens, extra=lead + 2)
    c.row_start += lead
    out, lse = c.run(tn, many=many)
    assert (out[:lead] == 7.5).all() and (lse[:lead] == 7.5).all(), "rows ahead of the first request were written"
    c.row_start -= lead
    c.q = _up(tn, c.q.numpy()[lead:], dtype)
    c.check((out[lead:], lse[lead:]))


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("H, G, rows, lens", [
    (2, 2, [300], [300]), (2, 4, [200, 90, 40], [1200, 1064, 90]), (1, 3, [1100], [1100]),
    (8, 8, [700, 600, 800], [1500, 1024, 800]),  # 256 rows a workgroup
])
def test_bf16_rows_of_up_to_1024_keys_have_them_exact(tn, D, H, G, rows, lens):
    """On the kernel of many rows, whose workgroups of rows past 1024 keys round them to f16: the lse of every row, on
    either side, within the bound of its side. Rows of few keys, whose lse is nearly a score, are among them."""
    c = Case(tn, "bfloat16", H, G, D, 32, rows, lens, seed=D)
    out, lse = c.run(tn, many=True)
    c.check((out, lse))
    ref = P.attend(c.q.numpy().astype(np.float64), c.cache, c.row_start, c.lens, c.table)
    keys = P.row_keys(c.row_start, c.lens, len(out))
    _, tol = P.tolerance("bfloat16", ref[0], ref[1], *ref[2:], c.max_len, D, rounded=keys > 1024, biased=False)
    few = np.repeat(np.array(rows) * G <= 128, rows)  # the kernel of few rows: keys exact, codes biased
    _, tol_few = P.tolerance("bfloat16", ref[0], ref[1], *ref[2:], c.max_len, D, rounded=False)
    worst = np.abs(lse - ref[1]) / np.where(few[:, None], tol_few, tol)
    print(f"  lse: up to 1024 keys {worst[keys <= 1024].max():.3f} of the bound, others "
          f"{worst[keys > 1024].max(initial=0):.3f}", flush=True)
    assert worst.max() <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D, S", [(64, 16), (128, 32), (192, 16)])
@pytest.mark.parametrize("rows, lens", [([1, 1, 3], [40, 700, 5]), ([90, 4, 130], [300, 1100, 130])])
@pytest.mark.parametrize("many", [False, True])
def test_queries_that_are_not_finite_reach_no_row_but_theirs(tn, many, dtype, D, S, rows, lens):
    """One element of a head's row NaN or infinite, and a row of nothing else: NaN out of it, every other row as exact
    as without it. Such rows lie in a wave with others and in a row's first, middle and last block."""
    c = Case(tn, dtype, 2, 3, D, S, rows, lens, seed=D)
    x = c.q.numpy().astype(np.float32)
    clean = x.copy()
    T = len(x)
    bad = {}
    for i, (what, e) in enumerate([(np.nan, 0), (np.inf, D - 1), (-np.inf, 33), (np.nan, D // 2), (None, 0)]):
        t, h = (i * 7) % T, (i * 5) % 6
        if (t, h) in bad:
            continue
        bad[t, h] = True
        if what is None:
            x[t, h] = np.where(np.arange(D) % 2, np.inf, np.nan)
        else:
            x[t, h, e] = what
    c.q = _up(tn, x, dtype)
    out, lse = c.run(tn, many=many)
    for t, h in bad:
        assert np.isnan(out[t, h]).all(), (t, h)
        assert not np.isposinf(lse[t, h]), (t, h)
    c.q = _up(tn, clean, dtype)
    want = c.run(tn, many=many)
    for t, h in bad:
        out[t, h], lse[t, h] = want[0][t, h], want[1][t, h]
    assert np.array_equal(out, want[0]) and np.array_equal(lse, want[1])
    c.check((out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, lens", [([3, 1, 5], [40, 700, 5]), ([90, 4, 130, 33], [300, 1100, 130, 2000])])
@pytest.mark.parametrize("most", [1, 2, 40])
@pytest.mark.parametrize("many", [False, True])
def test_rows_past_the_bound_are_not_computed(tn, many, most, dtype, rows, lens):
    """max_rows below a request's rows: its first ones as ever (their keys counted with all rows), the others left."""
    c = Case(tn, dtype, 2, 4, 64, 16, rows, lens, extra=2)
    out, lse = c.run(tn, many=many, max_rows=most)
    whole = c.run(tn, many=many)
    for r, n in enumerate(rows):
        a = c.row_start[r] + min(n, most)
        z = c.row_start[r + 1]
        assert (out[a:z] == 7.5).all() and (lse[a:z] == 7.5).all(), r
        out[a:z], lse[a:z] = whole[0][a:z], whole[1][a:z]
    c.check((out, lse))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, lens", [([3, 1, 5], [40, 700, 5]), ([90, 4, 130, 33], [300, 1100, 130, 2000])])
@pytest.mark.parametrize("most", [1, 33, 128, 1030])
def test_lengths_past_the_bound_are_cut_to_it(tn, most, dtype, rows, lens):
    """As a call of the shorter lengths, whose first rows may have no keys."""
    c = Case(tn, dtype, 2, 4, 64, 16, rows, lens, extra=2)
    got = c.run(tn, max_len=min(most, c.table.shape[1] * 16))  # (never past what the table holds)
    c.lens = [min(x, most) for x in lens]
    c.check(got)


@pytest.mark.parametrize("rows, lens", [([1, 2], [300, 40]), ([150], [150])])
@pytest.mark.parametrize("many", [False, True])
def test_f16_queries_below_the_normal_range(tn, many, rows, lens):
    """Multiples of 2^-24, f16's smallest number, with a scale that brings the scores back."""
    c = Case(tn, "float16", 2, 3, 64, 16, rows, lens, seed=4)
    c.q = _up(tn, c.q.numpy().astype(np.float32) * np.float32(2.0 ** -18), "float16")
    c.check(c.run(tn, scale=2.0 ** 15, many=many), scale=2.0 ** 15)


def _attend(tn, dev, dtype, q, T, Hq, D, row_start, lens, table, rows, most, out, lse):
    import ctypes

    from torchnative_amd import _lib as L

    t = [tn.tensor(np.ascontiguousarray(a, np.int32), device="hip") for a in (row_start, lens, table)]
    floats = dev.work_floats(len(lens), T, Hq, rows, most)
    work = tn.empty((floats + 1,), "float32", "hip")
    L.check(L.lib().tn_sdpa_paged_q4_0(
        None, ctypes.byref(dev._c), {"float32": 0, "bfloat16": 1, "float16": 2}[dtype], q.data_ptr(), Hq * D, T, Hq,
        len(lens), t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), np.shape(table)[1], rows, most, float("nan"),
        work.data_ptr(), floats, out.data_ptr(), lse.data_ptr()))
    tn.synchronize()


@pytest.mark.parametrize("rows, many", [(5, False), (200, True)])
def test_rows_and_outputs_past_two_to_the_31_elements(tn, rows, many):
    """The last rows of a call whose queries and outputs pass 4 GiB and 2^31 elements."""
    from test_paged_gpu import _fill
    from torchnative_amd import _lib as L

    c = Case(tn, "bfloat16", 2, 4, 256, 16, [rows], [rows + 300], seed=2)
    T = (1 << 20) + 37 + rows
    small = c.q.numpy().shape
    q, out = (tn.empty((T, 8, 256), "bfloat16", "hip") for _ in range(2))
    lse = tn.empty((T, 8), "float32", "hip")
    row = 8 * 256 * 2
    L.check(L.lib().tn_memcpy_d2d(q.data_ptr() + (T - rows) * row, c.q.data_ptr(), rows * row, None))
    guard = tn.tensor(np.full((64, 8, 256), 7.5, np.float32), dtype="bfloat16", device="hip")
    L.check(L.lib().tn_memcpy_d2d(out.data_ptr() + (T - rows - 64) * row, guard.data_ptr(), 64 * row, None))
    table = np.pad(c.table, ((0, 0), (0, 1 << 10)), constant_values=-1) if many else c.table
    most = table.shape[1] * 16 if many else c.max_len
    print("rows", rows, "of", T, flush=True)
    _attend(tn, _fill(tn, c.cache), "bfloat16", q, T, 8, 256, [T - rows, T], c.lens, table, rows, most, out, lse)
    got, glse = tn.empty((rows + 64, 8, 256), "bfloat16", "hip"), tn.empty((rows, 8), "float32", "hip")
    L.check(L.lib().tn_memcpy_d2d(got.data_ptr(), out.data_ptr() + (T - rows - 64) * row, (rows + 64) * row, None))
    L.check(L.lib().tn_memcpy_d2d(glse.data_ptr(), lse.data_ptr() + (T - rows) * 32, rows * 32, None))
    x = got.numpy().astype(np.float64)
    assert small == (rows, 8, 256) and (x[:64] == 7.5).all()
    c.check((x[64:], glse.numpy().astype(np.float64)))


def test_as_many_requests_as_a_call_takes(tn):
    """65535 requests of one row over one shared page, 1 to 16 tokens each: those of one length and query are equal, and
    the first of each right."""
    from test_paged_gpu import _fill

    n, D, Hq = 65535, 32, 2
    c = Case(tn, "float32", 1, 2, D, 16, [1] * 16, list(range(1, 17)), seed=9)
    for r in range(1, 16):  # one page for all
        c.table[r] = c.table[15]
    c.table[0] = c.table[15]
    r = np.arange(n) % 16
    q = _up(tn, c.q.numpy()[r], "float32")
    out, lse = tn.zeros((n, Hq, D)), tn.zeros((n, Hq))
    dev = _fill(tn, c.cache)
    _attend(tn, dev, "float32", q, n, Hq, D, np.arange(n + 1), r + 1, c.table[r], 1, 16, out, lse)
    x, y = out.numpy(), lse.numpy()
    assert np.array_equal(x, x[:16][r]) and np.array_equal(y, y[:16][r])
    c.check((x[:16].astype(np.float64), y[:16].astype(np.float64)))
