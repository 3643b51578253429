"""The 8-bit linear, the norms of heads and the paged 8-bit cache off the GPU: every refusal comes before a HIP call,
empty calls touch no pointer, and the oracle holds its own invariants."""

import ctypes
import os
import shutil

import numpy as np
import pytest

from oracle import int8 as I
from torchnative_amd import _lib
from torchnative_amd import hazard_scan as H

NAN = float("nan")


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


# --- rows in 8-bit integers and their product ------------------------------------------


def test_pitch(L):
    for k, want in ((1, 64), (63, 64), (64, 64), (65, 128), (576, 576), (4096, 4096), (0, 0), (-5, 0)):
        assert L.tn_i8_pitch(k) == want


def test_quantize_refusals(L):
    for dt in (_lib.TN_F64, _lib.TN_BOOL, 99):
        assert L.tn_i8_quantize(None, 16, dt, 1, 64, 16, 16) == _lib.TN_ENOTIMPL
        assert "float32, bfloat16 or float16" in _lib.last_error()
    assert L.tn_i8_quantize(None, 16, 0, 1, 0, 16, 16) == _lib.TN_EINVAL
    assert L.tn_i8_quantize(None, 16, 0, -1, 64, 16, 16) == _lib.TN_EINVAL
    assert L.tn_i8_quantize(None, 16, 0, 1, 131073, 16, 16) == _lib.TN_ENOTIMPL and "131073" in _lib.last_error()
    assert L.tn_i8_quantize(None, 16, 0, 1 << 24, 64, 16, 16) == _lib.TN_EVALUE
    for args in ((None, 16, 16), (16, None, 16), (16, 16, None)):
        assert L.tn_i8_quantize(None, args[0], 0, 1, 64, args[1], args[2]) == _lib.TN_EVALUE
        assert "null pointer" in _lib.last_error()
    assert L.tn_i8_quantize(None, 16, 0, 1, 64, 24, 16) == _lib.TN_EVALUE and "aligned" in _lib.last_error()
    assert L.tn_i8_quantize(None, None, 0, 0, 64, None, None) == _lib.TN_OK  # no rows: no pointer is touched


def test_matmul_and_linear_refusals(L):
    big = 1 << 40

    def mm(a=16, sa=16, m=2, k=64, w=16, sw=16, n=8, y=16, ydt=0):
        return L.tn_i8_matmul(None, a, sa, m, k, w, sw, n, None, y, ydt)

    def lin(x=16, dt=0, m=2, k=64, w=16, sw=16, n=8, work=16, size=big, y=16, ydt=0):
        return L.tn_i8_linear(None, x, dt, m, k, w, sw, n, None, work, size, y, ydt)

    for f in (mm, lin):
        for kw, code in (({"k": 0}, _lib.TN_EINVAL), ({"k": -64}, _lib.TN_EINVAL), ({"m": -1}, _lib.TN_EINVAL),
                         ({"n": -1}, _lib.TN_EINVAL), ({"k": 131073}, _lib.TN_ENOTIMPL), ({"m": 1 << 24}, _lib.TN_EVALUE),
                         ({"n": 1 << 24}, _lib.TN_EVALUE), ({"ydt": _lib.TN_F64}, _lib.TN_ENOTIMPL),
                         ({"w": None}, _lib.TN_EVALUE), ({"sw": None}, _lib.TN_EVALUE), ({"y": None}, _lib.TN_EVALUE),
                         ({"w": 8}, _lib.TN_EVALUE)):
            assert f(**kw) == code, (f, kw, _lib.last_error())
        assert f(k=0) == _lib.TN_EINVAL and "mat1 and mat2 shapes cannot be multiplied" in _lib.last_error()
        for kw in ({"m": 0}, {"n": 0}):
            assert f(w=None, y=None, **kw) == _lib.TN_OK
    assert mm(a=None) == _lib.TN_EVALUE and mm(sa=None) == _lib.TN_EVALUE and mm(a=8) == _lib.TN_EVALUE
    assert lin(x=None) == _lib.TN_EVALUE and lin(dt=_lib.TN_F64) == _lib.TN_ENOTIMPL
    for m in (1, 300):
        need = L.tn_i8_linear_work_bytes(m, 640)
        if need:
            assert lin(m=m, k=640, size=need - 1) == _lib.TN_EVALUE and f"needs {need}" in _lib.last_error()
            assert lin(m=m, k=640, work=None) == _lib.TN_EVALUE and lin(m=m, k=640, work=8) == _lib.TN_EVALUE
    assert L.tn_i8_linear_work_bytes(-1, 64) == 0 and L.tn_i8_linear_work_bytes(1, 0) == 0


def test_python_refusals():
    import torchnative_amd as tn

    x = tn.tensor(np.zeros((1, 64), np.float32))
    w = tn.I8Rows((8, 64), "cpu")
    assert w.codes.shape == (8, 64) and w.nbytes == 8 * 64 + 32 and tn.I8Rows((2, 65), "cpu").codes.shape == (2, 128)
    with pytest.raises(NotImplementedError, match="does not fall back to the host"):
        tn.i8_quantize(x)
    with pytest.raises(NotImplementedError, match="does not fall back to the host"):
        tn.i8_linear(x, w)
    with pytest.raises(TypeError, match="8-bit integers"):
        tn.i8_linear(x, x)
    with pytest.raises(TypeError, match="8-bit integers"):
        tn.i8_matmul(x, w)
    with pytest.raises(NotImplementedError, match="does not fall back to the host"):
        tn.qk_norm_rope(x, x, x, x, x, x)
    rows = tn.tensor(np.zeros((3, 6, 4), np.float32))
    for first, count in ((-1, 2), (5, 2), (0, 7), (0, -1)):
        with pytest.raises(RuntimeError, match="are not in rows"):
            tn.Heads(rows, first, count)
    h = tn.Heads(rows, 2, 3)
    assert h.shape == (3, 3, 4) and h.row_stride == 24 and h.dim() == 3


# --- norms and rotation -----------------------------------------------------------------


def test_heads_refusals(L):
    def call(dt=0, q=16, qs=256, Hq=4, k=16, ks=256, Hkv=2, m=2, d=64, qw=16, kw=16, f=16, rot=64, pos=16, qo=32,
             qos=256, ko=32, kos=256):
        return L.tn_qk_norm_rope(None, dt, q, qs, Hq, k, ks, Hkv, m, d, qw, kw, 1e-6, f, rot, pos, qo, qos, ko, kos)

    for kw, code in (({"dt": _lib.TN_F64}, _lib.TN_ENOTIMPL), ({"d": 0}, _lib.TN_ENOTIMPL), ({"d": 63}, _lib.TN_ENOTIMPL),
                     ({"d": 258}, _lib.TN_ENOTIMPL), ({"rot": 66}, _lib.TN_EINVAL), ({"rot": 31}, _lib.TN_EINVAL),
                     ({"rot": -2}, _lib.TN_EINVAL), ({"m": -1}, _lib.TN_EINVAL), ({"Hq": -1}, _lib.TN_EINVAL),
                     ({"Hkv": -1}, _lib.TN_EINVAL), ({"Hq": 65536, "qs": 1 << 30, "qos": 1 << 30}, _lib.TN_EVALUE),
                     ({"m": 1 << 31}, _lib.TN_EVALUE), ({"qs": 255}, _lib.TN_EINVAL), ({"kos": 127}, _lib.TN_EINVAL),
                     ({"ks": 1 << 62}, _lib.TN_EVALUE), ({"q": None}, _lib.TN_EVALUE), ({"ko": None}, _lib.TN_EVALUE),
                     ({"pos": None}, _lib.TN_EVALUE), ({"f": None}, _lib.TN_EVALUE), ({"qw": None}, _lib.TN_EVALUE),
                     ({"qo": 16, "qos": 300}, _lib.TN_EINVAL), ({"ko": 16, "kos": 300}, _lib.TN_EINVAL)):
        assert call(**kw) == code, (kw, _lib.last_error())
    assert call(m=0, q=None, pos=None) == _lib.TN_OK
    assert call(Hq=0, Hkv=0, pos=None) == _lib.TN_OK


def test_oracle_heads_against_complex_turns():
    """The rotation as a product of complex numbers, the norm by its definition."""
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((5, 3, 8)), rng.standard_normal(8)
    f, pos = np.array([1.0, 0.1, 0.01]), np.array([0, 1, 7, 1000, 3])
    got, _ = I.heads(x, w, f, pos, 1e-6)
    z = x / np.sqrt(np.mean(x ** 2, -1, keepdims=True) + 1e-6) * w
    turn = (z[..., :3] + 1j * z[..., 3:6]) * np.exp(1j * pos[:, None, None] * f)
    assert np.allclose(got[..., :3], turn.real) and np.allclose(got[..., 3:6], turn.imag)
    assert np.array_equal(got[..., 6:], z[..., 6:])


# --- the cache ----------------------------------------------------------------------------


def _cache(pages=8, size=16, heads=2, dim=64, planes=(16, 16, 16, 16)):
    return _lib.Q8Cache(*planes, pages, size, heads, dim)


@pytest.mark.parametrize("kw, code, word", [
    ({"size": 24}, _lib.TN_ENOTIMPL, "page_size 24"),
    ({"dim": 80}, _lib.TN_ENOTIMPL, "head_dim 80 is not implemented for a q8 cache"),
    ({"dim": 288}, _lib.TN_ENOTIMPL, "head_dim 288"),
    ({"heads": 0}, _lib.TN_EINVAL, "bad cache sizes"),
    ({"pages": -1}, _lib.TN_EINVAL, "bad cache sizes"),
    ({"pages": 1 << 27}, _lib.TN_EVALUE, "2^31 slots"),
    ({"planes": (16, 16, None, 16)}, _lib.TN_EVALUE, "null cache plane"),
    ({"planes": (16, 8, 16, 16)}, _lib.TN_EVALUE, "16-byte aligned"),
])
def test_cache_refusals_at_every_entry(L, kw, code, word):
    c = ctypes.byref(_cache(**kw))
    for st in (L.tn_kv_append_q8(None, c, _lib.TN_F32, 16, 16, 1, 4096, 16),
               L.tn_kv_read_q8(None, c, 16, 1, _lib.TN_F32, 16, 16),
               L.tn_sdpa_paged_q8(None, c, _lib.TN_F32, 16, 4096, 1, 4 * max(1, kw.get("heads", 2)), 1, 16, 16, 16, 4,
                                  1, 16, NAN, 16, 1 << 40, 16, 16)):
        assert st == code and word in _lib.last_error()
    for st in (L.tn_kv_append_q8(None, None, _lib.TN_F32, 16, 16, 1, 4096, 16),
               L.tn_kv_read_q8(None, None, 16, 1, _lib.TN_F32, 16, 16)):
        assert st == _lib.TN_EVALUE and "null cache" in _lib.last_error()


def test_row_refusals(L):
    c = ctypes.byref(_cache())
    for dt in (_lib.TN_F64, _lib.TN_BOOL, 99):
        assert L.tn_kv_append_q8(None, c, dt, 16, 16, 1, 128, 16) == _lib.TN_ENOTIMPL
        assert L.tn_kv_read_q8(None, c, 16, 1, dt, 16, 16) == _lib.TN_ENOTIMPL
    assert L.tn_kv_append_q8(None, c, 0, 16, 16, -1, 128, 16) == _lib.TN_EINVAL
    assert L.tn_kv_append_q8(None, c, 0, 16, 16, 2, 127, 16) == _lib.TN_EINVAL and "row stride" in _lib.last_error()
    assert L.tn_kv_append_q8(None, c, 0, 16, 16, 2, 1 << 62, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q8(None, c, 0, 16, 16, 1 << 31, 128, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q8(None, c, 0, None, 16, 1, 128, 16) == _lib.TN_EVALUE
    assert L.tn_kv_read_q8(None, c, 16, 1, 0, None, 16) == _lib.TN_EVALUE
    assert L.tn_kv_append_q8(None, c, 0, None, None, 0, 128, None) == _lib.TN_OK  # no rows: no pointer is touched
    assert L.tn_kv_read_q8(None, c, None, 0, 0, None, None) == _lib.TN_OK


def test_attention_refusals(L):
    c = ctypes.byref(_cache())

    def call(dtype=0, q=16, stride=256, tokens=2, Hq=4, n=1, starts=16, lens=16, table=16, width=4, rows=2, most=64,
             work=16, floats=1 << 40, out=16):
        return L.tn_sdpa_paged_q8(None, c, dtype, q, stride, tokens, Hq, n, starts, lens, table, width, rows, most, NAN,
                                  work, floats, out, None)

    assert call(dtype=_lib.TN_F64) == _lib.TN_ENOTIMPL
    assert call(Hq=5) == _lib.TN_ENOTIMPL and "do not divide" in _lib.last_error()
    for kw in ({"tokens": -1}, {"n": -1}, {"rows": -1}, {"most": -1}, {"Hq": -2}, {"width": -1}):
        assert call(**kw) == _lib.TN_EINVAL, kw
    assert call(most=65) == _lib.TN_EINVAL and "past what 4 pages hold" in _lib.last_error()
    assert call(stride=255) == _lib.TN_EINVAL and "row stride" in _lib.last_error()
    for kw in ({"n": 1 << 17}, {"tokens": 1 << 31}, {"tokens": 1 << 29}, {"stride": 1 << 62},
               {"width": 1 << 28, "most": (1 << 30) + 1}):
        assert call(**kw) == _lib.TN_EVALUE, kw
    for kw in ({"q": None}, {"out": None}, {"starts": None}, {"lens": None}, {"table": None}):
        assert call(**kw) == _lib.TN_EVALUE and "null pointer" in _lib.last_error(), kw
    need = L.tn_sdpa_paged_q8_work_floats(c, 1, 2, 4, 2, 4096)
    assert need > 0
    assert call(most=4096, width=256, floats=need - 1) == _lib.TN_EVALUE and "this call needs" in _lib.last_error()
    assert call(most=4096, width=256, work=None) == _lib.TN_EVALUE and call(most=4096, width=256, work=8) == _lib.TN_EVALUE
    empty = ctypes.byref(_cache(pages=0, planes=(None,) * 4))
    assert L.tn_sdpa_paged_q8(None, empty, 0, 16, 256, 2, 4, 1, 16, 16, 16, 4, 2, 64, NAN, 16, 1 << 40, 16, None) == \
        _lib.TN_EINVAL and "no pages" in _lib.last_error()
    for kw in ({"n": 0}, {"tokens": 0}, {"rows": 0}, {"Hq": 0}):
        assert call(q=None, out=None, **kw) == _lib.TN_OK, kw


def test_work_floats_serve_smaller_calls(L):
    """A buffer for a loop's largest step serves every smaller one."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        H, G, D = int(rng.choice([1, 2, 8])), int(rng.choice([1, 4, 7])), int(rng.choice([32, 64, 128]))
        c = ctypes.byref(_cache(pages=1000, size=16, heads=H, dim=D))
        big = [int(rng.integers(1, x)) for x in (40, 3000, 3000, 16000)]
        n, tokens, rows, most = big
        need = L.tn_sdpa_paged_q8_work_floats(c, n, tokens, H * G, rows, most)
        small = [int(rng.integers(1, x + 1)) for x in big]
        assert L.tn_sdpa_paged_q8_work_floats(c, small[0], small[1], H * G, small[2], small[3]) <= need, (big, small)


def test_oracle_blocks_keep_their_values_as_rows_join():
    """Half a step when written, half of each larger step more."""
    rng = np.random.default_rng(3)
    c = I.Cache(1, 16, 2, 32)
    x = rng.standard_normal((16, 2, 32)).astype(np.float32) * np.geomspace(0.1, 3, 16, dtype=np.float32)[:, None, None]
    off = np.zeros((16, 2))
    for t in range(16):
        was = c.scale["k"][0].copy()
        c.append(x[t:t + 1], x[t:t + 1], [t])
        s = c.scale["k"][0].astype(np.float64)
        off[:t] += np.where(s > was, s / 2 * 1.00001, 0)
        off[t] = s / 2 * 1.00001
        got = c.rows("k", np.arange(t + 1))
        assert (np.abs(got - x[:t + 1]) <= off[:t + 1, :, None] + 1e-6 * np.abs(x[:t + 1])).all()
    whole = I.Cache(1, 16, 2, 32)
    whole.append(x, x, np.arange(16))
    assert np.array_equal(whole.scale["k"], c.scale["k"])


@pytest.mark.skipif(shutil.which(H.build.HIPCC) is None and not os.path.exists(H.build.HIPCC),
                    reason="hipcc is not installed")
def test_ring_stages_of_the_products_are_read_before_they_are_opened(tmp_path):
    asm = H.assembly("i8.hip", str(tmp_path))
    for kernel in ("k_i8_gemm", "k_i8_large"):
        assert kernel in asm
        assert H.open_barriers(asm, kernel) == []


def test_rows_of_codes_refuse_planes_that_do_not_hold_them():
    from torchnative_amd import _C
    from torchnative_amd.tensor import Tensor

    def t(shape, dtype):
        return Tensor(shape, dtype, "cpu", _host=np.zeros(shape, dtype))

    rows = _C.I8Rows((3, 70), "cpu", t((3, 128), "int8"), t((3,), "float32"))
    assert rows.shape == (3, 70)
    for codes, scales in ((t((3, 70), "int8"), t((3,), "float32")), (t((2, 128), "int8"), t((3,), "float32")),
                          (t((3, 128), "uint8"), t((3,), "float32")), (t((3, 128), "int8"), t((2,), "float32")),
                          (t((3, 128), "int8"), t((3,), "float64"))):
        with pytest.raises(RuntimeError, match="do not hold rows"):
            _C.I8Rows((3, 70), "cpu", codes, scales)


def test_an_output_over_an_input_is_refused(L):
    """Workgroups would read what others have written: one byte in common is enough, none is not."""
    m, n, k = 3, 100, 200
    x, w, far = 1 << 20, 1 << 24, 1 << 28

    def lin(y, work=far, m=m):
        return L.tn_i8_linear(None, x, _lib.TN_BF16, m, k, w, far, n, None, work, 1 << 40, y, _lib.TN_F32)

    def mm(y):
        return L.tn_i8_matmul(None, x, far, m, k, w, far, n, None, y, _lib.TN_F32)

    ysize, pitch = m * n * 4, 256
    for f, size in ((lin, m * k * 2), (mm, m * pitch)):
        for y in (x, x + size - 4, x - ysize + 4, w, w + n * pitch - 4, w - ysize + 4):
            assert f(y) == _lib.TN_EINVAL and "y overlaps an input" in _lib.last_error(), (f, y)
    need = L.tn_i8_linear_work_bytes(300, k)
    for y in (far, far + need - 4):
        assert lin(y, m=300) == _lib.TN_EINVAL and "overlaps" in _lib.last_error()
