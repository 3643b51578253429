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
