"""Rows of the paged attention at the edges of a call: ahead of the first request's, past the bounds on rows and
lengths, queries that are not finite."""

import numpy as np
import pytest

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
