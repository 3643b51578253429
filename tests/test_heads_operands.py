"""Heads of stacked rows have a row stride of their own. An entry point either hands that stride on or refuses them: none
takes their pointer for dense rows. Run with a library that records its calls, so no GPU is needed."""

import ctypes
import sys

import pytest

import torchnative_amd as tn
from torchnative_amd import _C, _lib, nn, paged

T = sys.modules["torchnative_amd.tensor"]  # (the package's `tensor` is a function)


class _Buffer:
    ptr = 1 << 20


class _Recorder:
    """A library whose calls succeed and are kept."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call

    def named(self, name):
        return [a for n, a in self.calls if n == name]


@pytest.fixture
def calls(monkeypatch):
    rec = _Recorder()
    monkeypatch.setattr(T, "_DeviceBuffer", lambda nbytes: _Buffer())
    for mod in (T, _C, paged):
        monkeypatch.setattr(mod, "lib", lambda: rec)
    return rec


def _t(*shape, dtype="float32"):
    return tn.Tensor(shape, dtype, "hip")


def _heads():
    return tn.Heads(_t(5, 6, 64), 1, 4)


def _table():
    t = object.__new__(paged.PageTable)
    t.requests, t.width, t.page_size = 2, 4, 16
    t.row_start, t.lens, t.table = (_t(n, dtype="int32") for n in (3, 2, 8))
    return t


REFUSED = [
    ("sdpa_decode query", lambda h: tn.sdpa_decode(h, _t(5, 2, 8, 64), _t(5, 2, 8, 64), _t(5, dtype="int32"), 8)),
    ("i8_linear input", lambda h: tn.i8_linear(h, tn.I8Rows((7, 64)))),
    ("i8_linear out", lambda h: tn.i8_linear(_t(5, 4, 32), tn.I8Rows((64, 32)), out=h)),
    ("i8_matmul out", lambda h: tn.i8_matmul(tn.I8Rows((5, 32)), tn.I8Rows((64, 32)), out=h)),
    ("Int8Linear", lambda h: tn.Int8Linear(tn.I8Rows((7, 64)))(h)),
    ("i8_quantize", lambda h: tn.i8_quantize(h)),
    ("linear", lambda h: _C.linear(h, _t(7, 64))),
    ("nn.Linear", lambda h: nn.Linear(_t(7, 64))(h)),
    ("quantize", lambda h: tn._quantize(h, "q4_0")),
    ("attention", lambda h: tn.scaled_dot_product_attention(h, h, h)),
    ("mask", lambda h: tn.scaled_dot_product_attention(*(_t(4, 5, 4, 64) for _ in range(3)), attn_mask=h)),
    ("attend out, 4 bits", lambda h: tn.Q4Cache(8, 16, 2, 64).attend(_t(5, 4, 64), _table(), 5, 64, out=h)),
    ("attend out, 8 bits", lambda h: tn.Q8Cache(8, 16, 2, 64).attend(_t(5, 4, 64), _table(), 5, 64, out=h)),
    ("attend work", lambda h: tn.Q8Cache(8, 16, 2, 64).attend(_t(5, 4, 64), _table(), 5, 64, work=h)),
    ("append slots", lambda h: tn.Q8Cache(8, 16, 2, 64).append(_t(5, 2, 64), _t(5, 2, 64), h)),
    ("read slots", lambda h: tn.Q8Cache(8, 16, 2, 64).read(h)),
    ("rotation weights", lambda h: tn.qk_norm_rope(h, h, h, _t(64), _t(32), _t(5, dtype="int32"))),
]


@pytest.mark.parametrize("call", [c for _, c in REFUSED], ids=[n for n, _ in REFUSED])
def test_operands_taken_as_dense_rows_refuse_heads(calls, call):
    """attention's query fails an earlier check, of its four dims; everything else names the heads."""
    with pytest.raises((NotImplementedError, RuntimeError), match="dense rows|4 dims"):
        call(_heads())
    launched = [n for n, _ in calls.calls if n.startswith("tn_") and not n.endswith(("work_floats", "work_bytes"))]
    assert launched == []


def test_rows_with_a_stride_hand_it_on(calls):
    rows = _t(5, 8, 64)
    q, k, v = tn.Heads(rows, 0, 4), tn.Heads(rows, 4, 2), tn.Heads(rows, 6, 2)
    base = rows.data_ptr()
    tn.qk_norm_rope(q, k, _t(64), _t(64), _t(32), _t(5, dtype="int32"))
    (a,) = calls.named("tn_qk_norm_rope")
    assert (a[2], a[3], a[5], a[6]) == (base, 512, base + 4 * 64 * 4, 512) and (a[17], a[19]) == (512, 512)
    for cache, kind in ((tn.Q4Cache(8, 16, 2, 64), "q4_0"), (tn.Q8Cache(8, 16, 2, 64), "q8")):
        cache.append(k, v, _t(5, dtype="int32"))
        (a,) = calls.named(f"tn_kv_append_{kind}")
        assert a[3:7] == (base + 4 * 64 * 4, base + 6 * 64 * 4, 5, 512)
        cache.attend(q, _table(), 5, 64)
        (a,) = calls.named(f"tn_sdpa_paged_{kind}")
        assert a[3:5] == (base, 512)
    assert isinstance(cache._c, ctypes.Structure) and _lib.Q8Cache is type(cache._c)


def test_rows_of_codes_are_where_their_planes_are(calls):
    """Whatever the device is called, or not named at all."""
    for name in ("hip", "cuda", "cuda:0", "hip:0"):
        w = tn.I8Rows((7, 64), name)
        assert w.device == "hip"
        tn.i8_linear(_t(5, 64), w, out=_t(5, 7))
        assert calls.named("tn_i8_linear")[-1][5] == w.codes.data_ptr()
    host = [tn.Tensor(s, d, "cpu") for s, d in (((7, 64), "int8"), ((7,), "float32"))]
    assert tn.I8Rows((7, 64), codes=host[0], scales=host[1]).device == "cpu"
    with pytest.raises(RuntimeError, match="codes on cpu and scales on hip"):
        tn.I8Rows((7, 64), codes=host[0], scales=_t(7))
