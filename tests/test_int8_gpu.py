"""The 8-bit linear, the norms of heads and the paged 8-bit cache on the GPU against oracle/int8.py: integers, codes,
scales and the linear's outputs bit for bit, norms and attention within bounds derived from their roundings."""

import ctypes
import functools

import numpy as np
import pytest
from test_int8_shapes import PRODUCTS

from oracle import int8 as I
from oracle import paged as P

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]
CODE = {"float32": 0, "bfloat16": 1, "float16": 2}


@pytest.fixture(scope="module")
def tn():
    import torchnative_amd as tn

    print("device:", tn._hip_probe(), flush=True)
    return tn


def _up(tn, a, dtype=None):
    return tn.tensor(a, dtype=dtype, device="hip")


def _ints(tn, a):
    return tn.tensor(np.asarray(a, np.int32), device="hip")


def _narrow(tn, a, dtype):
    """f32 values rounded once to `dtype`, as bits."""
    if dtype == "float32":
        return np.asarray(a, np.float32)
    with np.errstate(over="ignore"):
        return tn.tensor(np.asarray(a, np.float32), dtype=dtype).bits()


# --- rows in 8-bit integers and their product ------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (3, 5), (2, 63), (4, 64), (5, 65), (7, 576), (1, 1024), (6, 1025), (3, 4095),
                                  (2, 4099), (2, 16384), (1, 131072), (200, 130)])
def test_quantize(tn, dtype, m, k):
    rng = np.random.default_rng(m + k)
    x = (rng.standard_normal((m, k)) * 10.0 ** rng.integers(-4, 3, (m, 1))).astype(np.float32)
    x[0, : k // 2] = 0
    x[-1] = np.float32(0) if m > 2 else x[-1]
    t = _up(tn, x, dtype)
    codes, scales = I.quantize(t.numpy().astype(np.float32))
    out = tn.I8Rows((m, k))
    from torchnative_amd import _lib as L

    L.check(L.lib().tn_memset(out.codes.data_ptr(), 0x55, out.codes.nbytes, None))
    got = tn.i8_quantize(t, out)
    pad = np.zeros((m, got.codes.shape[1]), np.int64)
    pad[:, :k] = codes
    assert np.array_equal(got.codes.numpy().astype(np.int64), pad)
    assert got.scales.numpy().tobytes() == scales.tobytes()


def test_quantize_of_ties_and_extremes(tn):
    """Halves to even; values at the scale's ends; rows of tiny, huge and not finite values."""
    x = np.zeros((9, 130), np.float32)
    x[0, :4] = [127, 0.5, 1.5, -2.5]
    x[1, :3] = [2.0 ** -140, -(2.0 ** -149), 2.0 ** -126]
    x[2, :3] = [3.0e38, -3.4e38, 1e30]
    x[3, 129] = np.inf
    x[4, 128] = np.nan
    x[5, 3], x[5, 77] = -np.inf, np.nan
    x[6] = np.linspace(-1, 1, 130)
    x[8, 64] = -5
    got = tn.i8_quantize(_up(tn, x))
    codes, scales = I.quantize(x)
    assert np.array_equal(got.codes.numpy()[:, :130].astype(np.int64), codes)
    assert got.scales.numpy().tobytes() == scales.tobytes()
    assert list(codes[0, :4]) == [127, 0, 2, -2] or list(codes[0, :4]) == [127, 0, 1, -2]
    w = tn.i8_quantize(_up(tn, np.ones((3, 130), np.float32)))
    y = tn.i8_linear(_up(tn, x), w).numpy()
    assert np.isnan(y[3:6]).all() and np.isfinite(y[[0, 1, 2, 6, 7, 8]]).all() and (y[7] == 0).all()


def _product(tn, m, n, k, seed, dtype="float32", odt="float32", bias=False, extreme=False):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((m, k)) * 10.0 ** rng.integers(-3, 3, (m, 1))).astype(np.float32)
    w = rng.standard_normal((n, k)).astype(np.float32) * np.float32(0.05)
    if extreme:  # every code +-127: the largest sums
        x, w = np.sign(x) * np.float32(2), np.sign(w) * np.float32(3)
        x[0], w[0] = 2, 3
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    tx = _up(tn, x, dtype)
    cx, sx = I.quantize(tx.numpy().astype(np.float32))
    cw, sw = I.quantize(w)
    want = _narrow(tn, I.linear(cx, sx, cw, sw, b), odt)
    tw = tn.i8_quantize(_up(tn, w))
    print(f"case [{m}, {k}] x [{n}, {k}] {dtype} -> {odt} bias {bias}", flush=True)
    got = tn.i8_linear(tx, tw, _up(tn, b) if bias else None, out_dtype=odt)
    bits = got.numpy() if odt == "float32" else got.bits()
    assert bits.tobytes() == want.tobytes(), np.argwhere(bits != want)[:5]
    # and against the product of the values themselves: each code is off by half a step
    x64, w64 = tx.numpy().astype(np.float64), w.astype(np.float64)
    ref = x64 @ w64.T + (0 if b is None else b)
    s, t = sx.astype(np.float64)[:, None] / 2 * 1.0001, sw.astype(np.float64)[None] / 2 * 1.0001
    bound = np.abs(x64).sum(1)[:, None] * t + np.abs(w64).sum(1)[None] * s + k * s * t
    step = {"float32": 2.0 ** -22, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[odt]
    assert (np.abs(got.numpy().astype(np.float64) - ref) <= bound + 2 * step * (np.abs(ref) + bound) + 1e-7).all()
    return tx, tw, bits


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 127, 129, 200, 257])
@pytest.mark.parametrize("n, k", [(1, 1), (15, 70), (16, 64), (130, 576), (257, 191), (300, 1024), (1536, 576)])
def test_linear(tn, m, n, k):
    _product(tn, m, n, k, m * n, DTYPES[(m + n) % 3], DTYPES[(m // 2 + k) % 3], bias=(m + k) % 2 == 0)


@pytest.mark.parametrize("m, n, k", [(1, 14336, 4096), (16, 4097, 4096), (512, 1000, 4096), (1, 5, 131072),
                                     (40, 3, 131072), (2049, 513, 320), (777, 5000, 128), (4096, 512, 64),
                                     (20, 20000, 72), (1000, 1024, 1000), (256, 256, 8192), (600, 768, 2112)])
@pytest.mark.parametrize("extreme", [False, True])
def test_linear_of_larger_sizes(tn, m, n, k, extreme):
    _product(tn, m, n, k, m + n, "bfloat16" if m % 2 else "float16", "float32", bias=True, extreme=extreme)


def test_a_rows_bits_do_not_depend_on_the_rows_around_it(tn):
    tx, tw, whole = _product(tn, 300, 700, 640, 5, "bfloat16", "bfloat16")
    x = tx.bits()
    for rows in (slice(0, 1), slice(7, 9), slice(100, 117), slice(30, 95), slice(0, 130)):
        part = tn.tensor(x[rows], dtype="bfloat16", device="hip")
        assert np.array_equal(tn.i8_linear(part, tw).bits(), whole[rows])
        assert np.array_equal(tn.i8_matmul(tn.i8_quantize(part), tw, out_dtype="bfloat16").bits(), whole[rows])


def test_linear_writes_nothing_else(tn):
    """Outputs inside a larger buffer, a work buffer of just its size, planes between others."""
    from torchnative_amd import _lib as L

    lib = L.lib()
    for m, n, k in ((1, 33, 100), (5, 70, 130), (37, 129, 200), (150, 300, 64)):
        for odt, size in (("float32", 4), ("bfloat16", 2)):
            rng = np.random.default_rng(m)
            x, w = (rng.standard_normal((r, k)).astype(np.float32) for r in (m, n))
            tx, tw = _up(tn, x), tn.i8_quantize(_up(tn, w))
            lead, need = 3, int(lib.tn_i8_linear_work_bytes(m, k))
            y = tn.tensor(np.full((lead + m * n + 5) * size, 0x5A, np.uint8), device="hip")
            work = tn.tensor(np.full(need + 64, 0x5A, np.uint8), device="hip")
            L.check(lib.tn_i8_linear(None, tx.data_ptr(), 0, m, k, tw.codes.data_ptr(), tw.scales.data_ptr(), n, None,
                                     work.data_ptr(), need, y.data_ptr() + lead * size, CODE[odt]))
            got = y.numpy()
            assert (got[: lead * size] == 0x5A).all() and (got[(lead + m * n) * size:] == 0x5A).all()
            assert (work.numpy()[need:] == 0x5A).all()
            want = tn.i8_linear(tx, tw, out_dtype=odt)
            want = want.numpy() if odt == "float32" else want.bits()
            assert got[lead * size: (lead + m * n) * size].tobytes() == want.tobytes()


def test_int8_layer_and_quantize_swap(tn):
    rng = np.random.default_rng(0)
    from torchnative_amd import nn

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.up = nn.Linear(rng.standard_normal((70, 33)).astype(np.float32), rng.standard_normal(70).astype(np.float32))
            self.down = nn.Linear(rng.standard_normal((33, 70)).astype(np.float32))

    model = Block()
    dense = {n: (m.weight.numpy(), m.bias.numpy() if m.bias else None) for n, m in model.named_children()}
    report = tn.quantize_(model, "i8")
    assert report.replaced == ["up", "down"] and report.quantized_bytes == 70 * 64 + 280 + 33 * 128 + 132
    x = rng.standard_normal((2, 3, 33)).astype(np.float32)
    y = model.up.to("cpu").to("hip")(_up(tn, x))
    assert y.shape == (2, 3, 70) and y.dtype == "float32"
    cx, sx = I.quantize(x.reshape(6, 33))
    want = I.linear(cx, sx, *I.quantize(dense["up"][0]), dense["up"][1])
    assert y.numpy().reshape(6, 70).tobytes() == want.tobytes()
    with pytest.raises(RuntimeError, match="cannot be multiplied"):
        model.down(_up(tn, x))


def test_linear_captured_and_replayed(tn):
    """Two graphs on two streams, each with a work buffer of its own, replayed side by side with eager calls between."""
    from torchnative_amd import _lib as L

    lib, runs = L.lib(), []
    for seed, (m, n, k) in enumerate(((1, 900, 576), (70, 640, 1000))):
        rng = np.random.default_rng(seed)
        x, w = (_up(tn, rng.standard_normal((r, k)).astype(np.float32)) for r in (m, n))
        w8 = tn.i8_quantize(w)
        want = tn.i8_linear(x, w8).numpy()
        need = int(lib.tn_i8_linear_work_bytes(m, k))
        work, y, s = tn.empty((need + 16,), "uint8"), tn.zeros((m, n)), tn.Stream()
        call = functools.partial(lib.tn_i8_linear, s.handle, x.data_ptr(), 0, m, k, w8.codes.data_ptr(),
                                 w8.scales.data_ptr(), n, None, work.data_ptr(), need, y.data_ptr(), 0)
        tn.synchronize()
        L.check(lib.tn_stream_begin_capture(s.handle))
        L.check(call())
        graph = ctypes.c_void_p()
        L.check(lib.tn_stream_end_capture(s.handle, ctypes.byref(graph)))
        runs.append((s, graph, y, want, call, (x, w8, work)))
    for rnd in range(4):
        for _, _, y, *_ in runs:
            y.zero_()
        tn.synchronize()
        for _ in range(5):
            for s, graph, *_ in runs:
                L.check(lib.tn_graph_launch(s.handle, graph))
        if rnd % 2:
            for *_, call, _ in runs:
                L.check(call())
        for s, _, y, want, *_ in runs:
            s.synchronize()
            assert np.array_equal(y.numpy(), want), rnd
    for _, graph, *_ in runs:
        L.check(lib.tn_graph_destroy(graph))


# --- norms of heads and their rotation --------------------------------------------------


def _heads_check(tn, dtype, x, w, f, pos, got, eps):
    ref, size = I.heads(x, w, f, pos, eps)
    tol = I.heads_tolerance(dtype, ref, size, x.shape[-1])
    worst = np.max(np.abs(got.astype(np.float64) - ref) / tol, initial=0)
    print(f"  worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, Hq, Hkv, d, rot", [
    (1, 9, 3, 64, 64), (3, 32, 8, 128, 128), (5, 4, 1, 128, 64), (2, 1, 1, 2, 2), (4, 3, 2, 6, 4), (7, 5, 5, 30, 0),
    (3, 8, 2, 80, 40), (2, 16, 0, 96, 96), (2, 0, 7, 192, 96), (3, 6, 2, 256, 256), (2, 3, 3, 250, 126), (2, 40, 8, 64, 16),
    (1025, 20, 4, 128, 128), (1300, 2, 1, 36, 20), (1100, 33, 32, 64, 32), (4, 2, 2, 160, 8), (3, 4, 4, 32, 32),
    (2, 5, 1, 254, 254), (1024, 17, 1, 256, 64)])
def test_heads(tn, dtype, m, Hq, Hkv, d, rot):
    rng = np.random.default_rng(m + d)
    q, k = ((rng.standard_normal((m, h, d)) * 10.0 ** rng.integers(-3, 3, (m, h, 1))).astype(np.float32) for h in (Hq, Hkv))
    qw, kw = (1 + 0.3 * rng.standard_normal(d).astype(np.float32) for _ in "qk")
    f = (1e5 ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32)
    pos = rng.integers(0, 40000, m).astype(np.int32)
    tq, tk, tf = _up(tn, q, dtype), _up(tn, k, dtype), _up(tn, f) if rot else tn.empty((0,), "float32")
    print(f"case {dtype} m {m} heads {Hq}/{Hkv} d {d} rot {rot}", flush=True)
    qo, ko = tn.empty(q.shape, dtype), tn.empty(k.shape, dtype)
    tn.qk_norm_rope(tq, tk, _up(tn, qw), _up(tn, kw), tf, _ints(tn, pos), 1e-5, qo, ko)
    for x, w, got in ((tq, qw, qo), (tk, kw, ko)):
        _heads_check(tn, dtype, x.numpy().astype(np.float64), w, f, pos, got.numpy(), 1e-5)
    before = [qo.bits(), ko.bits()]
    tn.qk_norm_rope(tq, tk, _up(tn, qw), _up(tn, kw), tf, _ints(tn, pos), 1e-5)  # in place
    assert np.array_equal(tq.bits(), before[0]) and np.array_equal(tk.bits(), before[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_at_far_positions(tn, dtype):
    """Angles to 2^31 turns' radians, both signs: no position loses the rotation's digits."""
    rng = np.random.default_rng(9)
    pos = np.array([0, 1, 131071, 1000000, 16777217, 2**31 - 1, -5, -(2**31)], np.int32)
    d = 64
    x = rng.standard_normal((len(pos), 3, d)).astype(np.float32)
    f = (1e4 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    one = np.ones(d, np.float32)
    q, k = _up(tn, x[:, :2], dtype), _up(tn, x[:, 2:], dtype)
    src = q.numpy().astype(np.float64)
    tn.qk_norm_rope(q, k, _up(tn, one), _up(tn, one), _up(tn, f), _ints(tn, pos))
    _heads_check(tn, dtype, src, one, f, pos, q.numpy(), 1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_heads_inside_stacked_rows_in_place(tn, dtype, lead):
    """q|k|v rows with a pitch and a start off any alignment: v, the gaps and the ends stay as they are."""
    from torchnative_amd import _lib as L

    rng = np.random.default_rng(lead)
    for m, Hq, Hkv, d in ((3, 4, 2, 64), (2, 3, 1, 128), (2, 2, 1, 48), (3, 2, 2, 10)):
        wide = (Hq + 2 * Hkv) * d + 5
        flat = rng.standard_normal(lead + m * wide + 3).astype(np.float32)
        x = _up(tn, flat, dtype)
        was, size = x.numpy().astype(np.float64), x.element_size
        w, f = 1 + 0.1 * rng.standard_normal(d).astype(np.float32), (100.0 ** -np.arange(d // 2)).astype(np.float32)
        pos = np.arange(5, 5 + m).astype(np.int32)
        qp, kp = x.data_ptr() + lead * size, x.data_ptr() + (lead + Hq * d) * size
        t = (_up(tn, w), _up(tn, f), _ints(tn, pos))
        L.check(L.lib().tn_qk_norm_rope(None, CODE[dtype], qp, wide, Hq, kp, wide, Hkv, m, d, t[0].data_ptr(),
                                        t[0].data_ptr(), 1e-6, t[1].data_ptr(), d, t[2].data_ptr(), qp, wide, kp, wide))
        got = x.numpy().astype(np.float64)
        at = lead + np.arange(m)[:, None] * wide + np.arange((Hq + Hkv) * d)
        rest = np.ones(flat.size, bool)
        rest[at.ravel()] = False
        assert np.array_equal(got[rest], was[rest])
        _heads_check(tn, dtype, was[at].reshape(m, Hq + Hkv, d), w, f, pos, got[at].reshape(m, Hq + Hkv, d), 1e-6)


def test_heads_of_zeros_infinities_and_nan(tn):
    x = np.zeros((4, 2, 8), np.float32)
    x[1, 0, 3], x[2, 1, 0], x[3, 0] = np.inf, np.nan, 1e25
    q = _up(tn, x)
    k = _up(tn, x[:, :1])
    one = _up(tn, np.ones(8, np.float32))
    tn.qk_norm_rope(q, k, one, one, _up(tn, np.array([1.0, 0.5], np.float32)), _ints(tn, [3, 4, 5, 6]))
    y = q.numpy()
    assert (y[0] == 0).all() and np.isnan(y[1, 0]).any() and np.isnan(y[2, 1]).all()
    assert (y[1, 1] == 0).all() and (y[2, 0] == 0).all() and np.isfinite(y[3, 1]).all()


# --- rows into the cache and back ------------------------------------------------------


def _put(tn, t, a):
    from torchnative_amd import _lib as L

    a = np.ascontiguousarray(a)
    assert a.nbytes == t.nbytes
    L.check(L.lib().tn_memcpy_h2d(t.data_ptr(), a.ctypes.data, a.nbytes, None))


def _fill(tn, c):
    """A device cache holding the oracle's planes."""
    d = tn.Q8Cache(c.P, c.S, c.H, c.D)
    for t, a in zip((d.k_codes, d.k_scales, d.v_codes, d.v_scales), c.planes()):
        _put(tn, t, a)
    return d


def _same_planes(d, c, note=""):
    got = [t.numpy().ravel() for t in (d.k_codes, d.k_scales, d.v_codes, d.v_scales)]
    for name, a, b in zip(("k_codes", "k_scales", "v_codes", "v_scales"), got, c.planes()):
        assert a.tobytes() == b.tobytes(), f"{note} {name}: {np.flatnonzero(a != b)[:8]}"


def _held(rng, P_, S, H, D):
    """A cache with random rows in every block."""
    c = I.Cache(P_, S, H, D)
    for w in "kv":
        c.code[w][:] = rng.integers(-127, 128, c.code[w].shape)
        c.scale[w][:] = (rng.random(c.scale[w].shape) / 40).astype(np.float32)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, D, S", [(1, 32, 16), (3, 64, 16), (2, 96, 32), (8, 128, 64), (1, 160, 128), (2, 192, 16),
                                     (3, 224, 32), (2, 256, 256)])
def test_append_writes_the_planes_and_read_gives_them_back(tn, dtype, H, D, S):
    rng = np.random.default_rng(D + S)
    P_ = 512 // S + 3
    c = _held(rng, P_, S, H, D)
    dev = _fill(tn, c)
    total = P_ * S
    # a prompt from the middle of a block on; single rows of many blocks; short runs; rows that are skipped; whole blocks
    many = np.concatenate([np.arange(b * 16 + o, b * 16 + min(16, o + n)) for b, o, n in
                           ((20, 3, 1), (4, 0, 16), (9, 15, 1), (11, 0, 1), (2, 7, 5), (17, 1, 15))])
    for step, slots in enumerate((np.arange(5, 5 + 301), rng.permutation(total // 16) * 16 + 9, many,
                                  np.array([-1, 40, 41, total, -2**31, 42, 2**31 - 1, 43]), np.arange(64, 96),
                                  np.array([33]), np.arange(100, 100 + 47), np.array([16, 0, 32]))):
        slots = slots.astype(np.int32)
        m = len(slots)
        x = [(rng.standard_normal((m, H, D)) * 10.0 ** rng.integers(-2, 2, (m, 1, 1))).astype(np.float32) for _ in "kv"]
        x[0][0] = 0
        k, v = (_up(tn, a, dtype) for a in x)
        print(f"case {dtype} H {H} D {D} S {S} step {step} rows {m}", flush=True)
        dev.append(k, v, _ints(tn, slots))
        c.append(k.numpy().astype(np.float32), v.numpy().astype(np.float32), slots)
        tn.synchronize()
        _same_planes(dev, c, f"step {step}")
        live = (slots >= 0) & (slots < total)
        look = np.concatenate([slots, rng.integers(0, total, 40)]).astype(np.int32)
        live = (look >= 0) & (look < total)
        for out in DTYPES:
            got = [t.bits() if out != "float32" else t.numpy() for t in dev.read(_ints(tn, look), out)]
            for w, y in zip("kv", got):
                code, scale = c.code[w][np.where(live, look, 0)], c.scale[w][np.where(live, look, 0) // 16]
                want = _narrow(tn, (code.astype(np.float32) * scale[..., None]).astype(np.float32), out)
                assert np.array_equal(y[live], want[live])
                vals = tn.tensor(y, dtype=out).numpy() if out != "float32" else y
                assert np.isnan(vals[~live]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1023, 1024, 1025, 1040, 3001])
def test_append_of_many_rows(tn, dtype, m):
    """Around where a wave takes a window of rows: prompts from every place of a block on, single rows among them."""
    rng = np.random.default_rng(m)
    H, D, S = 2, 64, 32
    c = _held(rng, 3 * m // S + 40, S, H, D)
    dev = _fill(tn, c)
    slots, at = [], 0
    while len(slots) < m:
        at += int(rng.integers(0, 20))
        n = int(rng.choice([1, 2, 15, 16, 17, 200]))
        slots += list(range(at, at + n))
        at = (at + n + 15) // 16 * 16
    slots = np.array(slots[:m], np.int32)
    slots[::97] = np.where(rng.random(len(slots[::97])) < 0.5, -1, slots[::97])
    assert slots.max() < c.P * S
    x = [_up(tn, rng.standard_normal((m, H, D)).astype(np.float32), dtype) for _ in "kv"]
    dev.append(*x, _ints(tn, slots))
    c.append(*(t.numpy().astype(np.float32) for t in x), slots)
    _same_planes(dev, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, m", [(1, 900), (2, 1025), (4, 1500), (4, 3001), (8, 3001)])
@pytest.mark.parametrize("order", ["runs", "any"])
def test_windows_of_one_to_sixteen_rows(tn, dtype, H, m, order):
    """A wave's window goes by rows and heads. Rows of a block as they come, or in any order, with holes and repeats;
    read back with repeats, runs and slots that are none, in every output type."""
    rng = np.random.default_rng(m + H)
    D, S = 96, 64
    P_ = m // S * 4 + 40
    c = _held(rng, P_, S, H, D)
    dev = _fill(tn, c)
    blocks, slots = rng.permutation(P_ * S // 16), []
    for b in blocks:
        n = int(rng.choice([1, 2, 9, 16]))
        if order == "runs":
            lo = int(rng.integers(0, 17 - n))
            rows = b * 16 + np.arange(lo, lo + n)
        else:
            rows = np.where(rng.random(n) < 0.2, -1, b * 16 + rng.integers(0, 16, n))
        slots += [int(x) for x in rows]
    assert len(slots) >= m
    slots = np.array(slots[:m], np.int32)
    x = [_up(tn, rng.standard_normal((m, H, D)).astype(np.float32), dtype) for _ in "kv"]
    print(f"case {dtype} H {H} rows {m} {order}", flush=True)
    dev.append(*x, _ints(tn, slots))
    c.append(*(t.numpy().astype(np.float32) for t in x), slots)
    _same_planes(dev, c)
    total = P_ * S
    look = np.concatenate([slots, slots[::-1], np.repeat(slots[:40], 5), np.arange(100, 400), [total, -7, 2**31 - 1]])
    look = look.astype(np.int32)[: m + 500]
    live = (look >= 0) & (look < total)
    for out in DTYPES:
        for w, t in zip("kv", dev.read(_ints(tn, look), out)):
            at = np.where(live, look, 0)
            want = (c.code[w][at].astype(np.float32) * c.scale[w][at // 16][..., None]).astype(np.float32)
            got = t.bits() if out != "float32" else t.numpy()
            assert np.array_equal(got[live], _narrow(tn, want, out)[live])
            assert np.isnan(t.numpy()[~live]).all()


def test_append_in_any_order_within_a_block_with_holes_and_repeats(tn):
    rng = np.random.default_rng(7)
    H, D = 2, 96
    c = _held(rng, 6, 32, H, D)
    dev = _fill(tn, c)
    for slots in ([7, 3, 5, 4], [40, 40, 41, 40, -1, 33], [19, -1, -1, 17, -1, 16, 18], list(range(79, 63, -1)),
                  [100, 3, 101, 5, 102, 100, 3, 99, 4], [160, 161, 170, 161, 192, 175, 162, -5, 160, 191, 160],
                  [21] * 16, [96, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, 97]):
        m = len(slots)
        x = [(rng.standard_normal((m, H, D)) * 10.0 ** rng.integers(-2, 1, (m, 1, 1))).astype(np.float32) for _ in "kv"]
        dev.append(*(_up(tn, a) for a in x), _ints(tn, slots))
        c.append(*x, slots)
        _same_planes(dev, c, str(slots))


def test_append_token_by_token_as_a_block_fills(tn):
    """The scale grows and the codes are rounded anew, as the oracle's do; a second pass over the block begins it anew."""
    rng = np.random.default_rng(1)
    c = I.Cache(2, 16, 3, 64)
    dev = _fill(tn, c)
    for rnd in range(2):
        for t in range(32):
            x = [(rng.standard_normal((1, 3, 64)) * rng.choice([0.01, 1, 30])).astype(np.float32) for _ in "kv"]
            dev.append(*(_up(tn, a) for a in x), _ints(tn, [t]))
            c.append(*x, [t])
            _same_planes(dev, c, f"round {rnd} token {t}")


def test_append_of_infinities_nan_and_scales_that_are_no_numbers(tn):
    x = np.zeros((4, 2, 32), np.float32)
    x[0, 0, :4] = [3e38, -np.inf, 1e6, 7]
    x[1, 0] = np.nan
    x[1, 1, ::2] = np.inf
    x[2, 1] = np.linspace(-1e-39, 1e-39, 32)
    x[3, 0, 5] = -3.4e38
    c = I.Cache(2, 16, 2, 32)
    c.scale["k"][0], c.scale["v"][0] = np.float32(np.nan), np.float32(np.inf)
    c.scale["k"][1], c.scale["v"][1] = np.float32(-1), np.float32(0)
    dev = _fill(tn, c)
    slots = [4, 5, 6, 7]
    for slots in ([4, 5, 6, 7], [20, 21, 22, 23], [0, 1, 2, 3], [8, 16, 17, 31]):
        dev.append(_up(tn, x), _up(tn, x[::-1].copy()), _ints(tn, slots))
        c.append(x, x[::-1], slots)
        _same_planes(dev, c, str(slots))
    assert all(np.isfinite(t.numpy()).all() for t in dev.read(_ints(tn, np.arange(32))))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_parts_of_stacked_rows_at_any_alignment(tn, dtype):
    from torchnative_amd import _lib as L

    rng = np.random.default_rng(4)
    m, H, D, lead = 21, 2, 64, 3
    wide = 4 * H * D + 5  # q|k|v rows with an odd pitch
    x = _up(tn, rng.standard_normal(lead + m * wide).astype(np.float32), dtype)
    c = _held(rng, 3, 16, H, D)
    dev = _fill(tn, c)
    slots = np.arange(5, 5 + m).astype(np.int32)
    size, ko, vo = x.element_size, lead + 2 * H * D, lead + 3 * H * D
    L.check(L.lib().tn_kv_append_q8(None, ctypes.byref(dev._c), CODE[dtype], x.data_ptr() + ko * size,
                                    x.data_ptr() + vo * size, m, wide, _ints(tn, slots).data_ptr()))
    tn.synchronize()
    h = x.numpy().astype(np.float32)
    rows = lambda o: np.stack([h[o + t * wide: o + t * wide + H * D] for t in range(m)]).reshape(m, H, D)  # noqa: E731
    c.append(rows(ko), rows(vo), slots)
    _same_planes(dev, c)
    # and as heads of rows [m, heads, D]
    t = _up(tn, rng.standard_normal((m, 4 * H, D)).astype(np.float32), dtype)
    dev.append(tn.Heads(t, 2 * H, H), tn.Heads(t, 3 * H, H), _ints(tn, slots))
    c.append(t.numpy()[:, 2 * H:3 * H].astype(np.float32), t.numpy()[:, 3 * H:].astype(np.float32), slots)
    _same_planes(dev, c)


# --- attention --------------------------------------------------------------------------


class Case:
    """Requests with rows[r] rows and lens[r] cached tokens, their pages at random; codes outside of a request's tokens
    are 127 under scales that are NaN."""

    def __init__(self, tn, dtype, H, G, D, S, rows, lens, seed=0, extra=0, spread=1.0, uneven=False):
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
        c = I.Cache(len(pages), S, H, D)
        for w in "kv":
            c.code[w][:], c.scale[w][:] = 127, np.float32(np.nan)
        for r, x in enumerate(lens):
            t = np.arange(x)
            slots = self.table[r, t // S] * S + t % S if x else np.zeros(0, np.int64)
            blocks = np.unique(slots // 16)
            for w in "kv":
                s = (0.5 + rng.random((len(blocks), H))) / 36 * spread
                if uneven:  # scales of blocks far apart, some of them 0
                    s *= 10.0 ** rng.integers(-4, 3, s.shape) * (rng.random(s.shape) > 0.1)
                c.scale[w][blocks] = s.astype(np.float32)
                c.code[w][slots] = np.clip(np.rint(rng.standard_normal((x, H, D)) * 36), -127, 127)
        self.cache = c
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        T = int(self.row_start[-1]) + extra
        self.q = _up(tn, rng.standard_normal((T, self.Hq, D)).astype(np.float32), dtype)
        self.max_rows, self.max_len = max(rows + [0]), max(lens + [0])

    def run(self, tn, dev=None, stream=None, scale=None, fill=7.5, lse=True, table=None, max_len=None, max_rows=None,
            bits=False, many=False, q=None, q_stride=None):
        """many: the bound of a length is so loose that the call is one of many products."""
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
              f"{self.lens} work {floats} many {many}", flush=True)
        L.check(L.lib().tn_sdpa_paged_q8(
            stream, ctypes.byref(dev._c), CODE[self.dtype], self.q.data_ptr() if q is None else q,
            q_stride or self.Hq * self.D, T, self.Hq, n, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(),
            table.shape[1], rows, most, float("nan") if scale is None else scale, work.data_ptr(), floats,
            out.data_ptr(), ls.data_ptr() if lse else None))
        tn.synchronize()
        if bits:
            return out.bits(), ls.bits()
        return out.numpy().astype(np.float64), ls.numpy().astype(np.float64)

    def check(self, got, scale=None, table=None, fill=7.5):
        out, lse = got
        ref = P.attend(self.q.numpy().astype(np.float64), self.cache, self.row_start, self.lens,
                       self.table if table is None else table, scale)
        ro, rl, pav, _, qk, _ = ref
        keys = max(self.max_len, 1)
        with np.errstate(invalid="ignore"):
            tol, ltol = I.tolerance(self.dtype, np.nan_to_num(ro), rl, np.nan_to_num(pav), np.nan_to_num(qk), keys,
                                    self.D, self.cache.value_size())
        own = np.zeros(len(out), bool)
        own[: self.row_start[-1]] = True
        assert (out[~own] == fill).all() and (lse[~own] == fill).all(), "rows behind the last request were written"
        dead = np.isnan(ro)
        assert np.array_equal(np.isnan(out[own]), dead[own])
        assert np.array_equal(np.isnan(lse[own]), np.isnan(rl[own]))
        fin = np.isfinite(rl)
        good = own & ~np.isnan(rl).any(1)
        assert np.array_equal(lse[good] == -np.inf, rl[good] == -np.inf)
        with np.errstate(invalid="ignore"):
            worst = np.max(np.where(own[:, None, None] & ~dead, np.abs(out - ro) / tol, 0), initial=0)
            lworst = np.max(np.where(own[:, None] & fin, np.abs(lse - rl) / ltol, 0), initial=0)
        print(f"  worst {worst:.3f} of the bound, lse {lworst:.3f}", flush=True)
        assert worst <= 1 and lworst <= 1, (worst, lworst)


MANY = pytest.mark.parametrize("many", [False, True])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(3, 3, 64, 16), (2, 4, 128, 16), (1, 1, 32, 32), (1, 7, 96, 64), (2, 8, 256, 128),
                                        (1, 2, 160, 16), (1, 3, 192, 256), (1, 5, 224, 32), (1, 20, 64, 16),
                                        (1, 16, 128, 32)])
def test_single_tokens(tn, dtype, H, G, D, S):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 200]
    c = Case(tn, dtype, H, G, D, S, [1] * len(lens), lens, seed=D, extra=2)
    c.check(c.run(tn))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D, G, lens", [(64, 3, [3000]), (128, 4, [1, 2500, 700]), (96, 1, [1999, 4]), (256, 2, [1100, 3])])
def test_single_tokens_over_long_contexts(tn, dtype, D, G, lens):
    c = Case(tn, dtype, 2, G, D, 16, [1] * len(lens), lens, seed=D)
    c.check(c.run(tn))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(3, 3, 64, 16), (2, 4, 128, 64), (1, 6, 96, 16), (1, 1, 256, 32), (1, 2, 32, 16),
                                        (1, 2, 160, 16), (1, 1, 192, 32), (1, 1, 224, 16)])
@pytest.mark.parametrize("rows, lens", [
    ([130], [130]), ([3, 0, 70, 1], [90, 40, 70, 200]), ([2, 5, 4], [300, 5, 65]), ([33, 257], [33, 300]),
])
@MANY
def test_chunks_and_whole_prompts(tn, many, dtype, H, G, D, S, rows, lens):
    c = Case(tn, dtype, H, G, D, S, rows, lens, seed=D + len(rows), extra=3)
    c.check(c.run(tn, many=many))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, G, D, S", [(2, 3, 64, 16), (1, 4, 128, 32), (1, 2, 96, 16), (1, 1, 256, 64), (1, 2, 32, 16)])
@pytest.mark.parametrize("rows, lens", [([90], [2100]), ([200, 1, 0, 70, 3], [1500, 900, 40, 70, 1033])])
@MANY
def test_chunks_behind_long_contexts(tn, many, dtype, H, G, D, S, rows, lens):
    """Keys split over workgroups, with rows whose part of the keys is empty."""
    c = Case(tn, dtype, H, G, D, S, rows, lens, seed=D + len(rows), extra=2)
    c.check(c.run(tn, many=many))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("rows", [[250, 1, 600, 0, 700, 513], [150, 1, 300, 0, 350, 199]])
def test_many_rows_of_many_heads(tn, dtype, D, rows):
    """More than 65536 folded rows, with a request of few rows among the others; and a little fewer."""
    c = Case(tn, dtype, 8, 8, D, 32, rows, [260, 500, 610, 3, 690, 513], seed=D)
    c.check(c.run(tn, many=True))


@pytest.mark.parametrize("dtype", DTYPES)
@MANY
def test_rows_without_keys_and_empty_requests(tn, many, dtype):
    """More rows than tokens: the first attend nothing. Requests of no rows, of no tokens, and of neither."""
    c = Case(tn, dtype, 2, 2, 64, 16, [5, 1, 0, 0, 40, 20], [2, 0, 33, 0, 17, 0], extra=1)
    got = c.run(tn, many=many)
    c.check(got)
    assert np.isnan(got[0][:3]).all() and (got[1][:3] == -np.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[1, 1, 2], [40, 3, 200], [300]])
@MANY
def test_rows_past_the_calls_are_cut(tn, many, dtype, rows):
    """row_start from below zero to past the last row is as if it ran from zero to it."""
    c = Case(tn, dtype, 2, 2, 64, 16, rows, [x + 70 for x in rows])
    c.row_start[0], c.row_start[-1] = -5, c.row_start[-1] + 1000
    got = c.run(tn, many=many)
    c.row_start[0], c.row_start[-1] = 0, c.q.shape[0]
    c.check(got)


@pytest.mark.parametrize("lens", [[70, 90], [1500, 2000]])
@pytest.mark.parametrize("rows", [[1, 3], [40, 90]])
@MANY
def test_rows_ahead_of_the_first_request_stay(tn, many, rows, lens):
    c = Case(tn, "bfloat16", 2, 2, 64, 16, rows, lens, extra=4)
    c.row_start += 3
    out, lse = c.run(tn, many=many)
    assert (out[:3] == 7.5).all() and (lse[:3] == 7.5).all() and (out[-1] == 7.5).all()
    assert np.isfinite(out[3:-1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 90])
@MANY
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
@MANY
def test_scales_of_any_sign_and_peaked_rows(tn, many, dtype, rows, scale):
    c = Case(tn, dtype, 2, 3, 64, 16, [rows, rows], [150, 75], seed=5)
    c.check(c.run(tn, scale=scale, many=many), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 75])
@pytest.mark.parametrize("spread", [1e-4, 300.0, 10000.0])
@MANY
def test_small_and_large_values(tn, many, dtype, rows, spread):
    c = Case(tn, dtype, 1, 4, 128, 32, [rows], [180], seed=6, spread=spread)
    scale = 0.1 / spread if spread > 1 else None
    c.check(c.run(tn, scale=scale, many=many), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, lens", [([1, 1], [700, 300]), ([75], [180]), ([300, 2], [900, 40])])
@MANY
def test_blocks_of_unlike_scales(tn, many, dtype, rows, lens):
    """Scales of keys and values from block to block by powers of ten, and zeros."""
    c = Case(tn, dtype, 2, 2, 64, 16, rows, lens, seed=11, uneven=True)
    c.check(c.run(tn, scale=0.01, many=many), scale=0.01)


@pytest.mark.parametrize("spread", [1e-30, 1e30])
@MANY
def test_values_far_outside_of_f16(tn, many, spread):
    for rows in (1, 90):
        c = Case(tn, "float32", 1, 2, 64, 16, [rows], [200], seed=12)
        for r in c.cache.scale["v"]:
            r *= np.float32(spread)
        c.check(c.run(tn, many=many))


@MANY
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
@MANY
def test_queries_that_are_not_finite_stay_among_themselves(tn, many, dtype):
    c = Case(tn, dtype, 1, 2, 64, 16, [40], [100], seed=2)
    clean = c.run(tn, bits=True, many=many)
    x = c.q.numpy().astype(np.float32)
    x[3, 1, 5], x[20, 0, 63], x[39, 1, 0] = np.nan, np.inf, -np.inf
    c.q = _up(tn, x, dtype)
    got = c.run(tn, bits=True, many=many)
    hit = np.zeros((40, 2), bool)
    hit[3, 1] = hit[20, 0] = hit[39, 1] = True
    assert np.array_equal(got[0][~hit], clean[0][~hit]) and np.array_equal(got[1][~hit], clean[1][~hit])
    assert np.isnan(c.run(tn, many=many)[0][hit]).all()


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
@MANY
def test_the_same_bits_every_time(tn, many, rows):
    c = Case(tn, "bfloat16", 2, 4, 128, 16, rows, [900, 1300, 40])
    first = c.run(tn, bits=True, many=many)
    for _ in range(3):
        again = c.run(tn, bits=True, many=many)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("rows", [[1, 1], [64, 3]])
def test_loose_bounds_and_bounds_that_cut(tn, rows):
    c = Case(tn, "float16", 1, 4, 64, 16, rows, [100, 130])
    c.check(c.run(tn, max_len=(c.table.shape[1]) * 16, max_rows=500))
    if rows[0] == 64:  # rows past max_rows stay
        out, _ = c.run(tn, max_rows=10)
        assert (out[10:64] == 7.5).all() and np.isfinite(out[:10]).all() and np.isfinite(out[64:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 66])
@MANY
def test_query_rows_inside_stacked_rows(tn, many, dtype, rows):
    c = Case(tn, dtype, 2, 2, 96, 16, [rows, rows], [70, 130])
    want = c.run(tn, bits=True, many=many)
    T, Hq, D = c.q.shape
    wide, lead = Hq * D + 7, 5
    x = np.full(lead + T * wide, np.nan, np.float32)
    for t in range(T):
        x[lead + t * wide: lead + t * wide + Hq * D] = c.q.numpy()[t].ravel()
    x = _up(tn, x, dtype)
    got = c.run(tn, bits=True, many=many, q=x.data_ptr() + lead * x.element_size, q_stride=wide)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_a_cache_past_four_gigabytes(tn):
    """Pages whose bytes lie behind 2^32: the same result as from the first pages."""
    H, D, S = 8, 256, 256
    pages = (1 << 32) // (H * S * D) + 40
    for many in (False, True):
        small = Case(tn, "bfloat16", H, 1, D, S, [1, 90], [700, 300], seed=3)
        far, near = tn.Q8Cache(pages, S, H, D), _fill(tn, small.cache)
        from torchnative_amd import _lib as L

        shift = pages - small.cache.P
        for a, b in zip((near.k_codes, near.k_scales, near.v_codes, near.v_scales),
                        (far.k_codes, far.k_scales, far.v_codes, far.v_scales)):
            L.check(L.lib().tn_memcpy_d2d(b.data_ptr() + b.nbytes - a.nbytes, a.data_ptr(), a.nbytes, None))
        table = np.where(small.table >= 0, small.table + shift, -1)
        want = small.run(tn, dev=near, bits=True, many=many)
        got = small.run(tn, dev=far, table=table, bits=True, many=many)
        assert all(np.array_equal(a, b) for a, b in zip(want, got))
    # and rows written there
    rng = np.random.default_rng(1)
    k, v = (_up(tn, rng.standard_normal((5, H, D)).astype(np.float32)) for _ in range(2))
    at = np.array([pages * S - 16, pages * S - 15, (pages - 1) * S, shift * S + 32, shift * S + 33], np.int32)
    far.append(k, v, _ints(tn, at))
    near.append(k, v, _ints(tn, at - shift * S))
    for a, b in zip(far.read(_ints(tn, at)), near.read(_ints(tn, at - shift * S))):
        assert np.array_equal(a.numpy(), b.numpy()) and np.isfinite(a.numpy()).all()


# --- a run of them together ------------------------------------------------------------------


class Block:
    """An attention block held in 8 bits, as a program runs it: the stacked projection, the norms of heads with their
    rotation in place, the cache, the attention, the output projection. Everything it needs stays on the device."""

    def __init__(self, tn, dtype, hidden, H, G, D, requests, tokens, S, width, pages, seed):
        rng = np.random.default_rng(seed)
        self.tn, self.dtype, self.H, self.Hq, self.D, self.tokens, self.most = tn, dtype, H, H * G, D, tokens, width * S
        self.w = {n: rng.standard_normal(s).astype(np.float32) * np.float32(0.05) for n, s in
                  (("qkv", ((G + 2) * H * D, hidden)), ("o", (hidden, H * G * D)))}
        self.norm = {n: 1 + 0.2 * rng.standard_normal(D).astype(np.float32) for n in "qk"}
        self.freq = (1e4 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
        from torchnative_amd import nn

        self.qkv, self.o = (tn.Int8Linear.from_linear(nn.Linear(self.w[n])) for n in ("qkv", "o"))
        self.dev = {n: _up(tn, a) for n, a in (("q", self.norm["q"]), ("k", self.norm["k"]), ("f", self.freq))}
        self.table = tn.PageTable(requests, width, S, pages, tokens)
        self.cache = tn.Q8Cache(pages, S, H, D)
        self.x = tn.zeros((tokens, hidden), dtype)
        self.rows = tn.zeros((tokens, (G + 2) * H, D), dtype)
        self.a, self.lse = tn.zeros((tokens, self.Hq, D), dtype), tn.zeros((tokens, self.Hq))
        self.y = tn.zeros((tokens, hidden), dtype)
        from torchnative_amd import _lib as L

        lib = L.lib()
        self.works = [tn.empty((int(lib.tn_i8_linear_work_bytes(tokens, k)) + 16,), "uint8") for k in (hidden, self.Hq * D)]
        self.work = tn.empty((self.cache.work_floats(requests, tokens, self.Hq, tokens, self.most) + 1,), "float32")

    def step(self):
        tn, H, Hq = self.tn, self.H, self.Hq
        flat = self.rows.view(self.tokens, (Hq + 2 * H) * self.D)
        self.table.step()
        self.qkv(self.x, work=self.works[0], out=flat)
        q, k, v = tn.Heads(self.rows, 0, Hq), tn.Heads(self.rows, Hq, H), tn.Heads(self.rows, Hq + H, H)
        tn.qk_norm_rope(q, k, self.dev["q"], self.dev["k"], self.dev["f"], self.table.pos)
        self.cache.append(k, v, self.table.slots)
        self.cache.attend(q, self.table, self.tokens, self.most, work=self.work, out=self.a, lse=self.lse)
        self.o(self.a.view(self.tokens, Hq * self.D), work=self.works[1], out=self.y)


def _loop(tn, dtype, steps, capture, seed=0):
    """A serving loop of prompts and single tokens, ended requests and new ones, checked stage by stage."""
    from torchnative_amd import _lib as L

    lib = L.lib()
    n, H, G, D, S, width, pages, tokens, hidden = 4, 2, 3, 64, 16, 8, 24, 96, 200
    b = Block(tn, dtype, hidden, H, G, D, n, tokens, S, width, pages, seed)
    rng, s = np.random.default_rng(seed + 1), tn.Stream()
    for t in (b.cache.k_codes, b.cache.k_scales, b.cache.v_codes, b.cache.v_scales):  # pages that nothing was written to
        L.check(lib.tn_memset(t.data_ptr(), 0x80, t.nbytes, None))
    tn.synchronize()
    c = I.Cache(pages, S, H, D)
    o = {"lens": np.zeros(n, np.int32), "table": np.full((n, width), -1, np.int32),
         "free": np.arange(pages, dtype=np.int32)[::-1].copy(), "state": np.array([pages, 0], np.int32)}
    graph = None
    with s:
        if capture:
            L.check(lib.tn_stream_begin_capture(s.handle))
            b.step()
            graph = ctypes.c_void_p()
            L.check(lib.tn_stream_end_capture(s.handle, ctypes.byref(graph)))
        for i, fresh in enumerate(steps):
            x = tn.tensor(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype=dtype)
            for t, a in ((b.table.fresh, np.asarray(fresh, np.int32)), (b.x, x.bits())):
                a = np.ascontiguousarray(a)
                L.check(lib.tn_memcpy_h2d(t.data_ptr(), a.ctypes.data, a.nbytes, s.handle))
            if capture:
                L.check(lib.tn_graph_launch(s.handle, graph))
            else:
                b.step()
            s.synchronize()
            o = P.plan(np.asarray(fresh, np.int32), o["lens"], o["table"], S, o["free"], o["state"], tokens)
            assert np.array_equal(b.table.lens.numpy(), o["lens"]) and np.array_equal(b.table.slots.numpy(), o["slots"])
            # the projection, bit for bit up to the norms' input; v stays as it left it
            cx, sx = I.quantize(x.numpy().astype(np.float32))
            proj = tn.tensor(I.linear(cx, sx, *I.quantize(b.w["qkv"])), dtype=dtype)
            pv = proj.numpy().astype(np.float64).reshape(tokens, -1, D)
            rows = b.rows.numpy().astype(np.float64)
            assert np.array_equal(rows[:, b.Hq + H:], pv[:, b.Hq + H:]), f"step {i}"
            for lo, hi, w in ((0, b.Hq, b.norm["q"]), (b.Hq, b.Hq + H, b.norm["k"])):
                _heads_check(tn, dtype, pv[:, lo:hi], w, b.freq, o["pos"], rows[:, lo:hi], 1e-6)
            # the cache, from the rows that are there
            f32 = rows.astype(np.float32)
            c.append(f32[:, b.Hq:b.Hq + H], f32[:, b.Hq + H:], o["slots"])
            live = o["slots"] >= 0
            for w, t in zip("kv", b.cache.read(_ints(tn, o["slots"][live]))):
                got = c.code[w][o["slots"][live]].astype(np.float32) * c.scale[w][o["slots"][live] // 16][..., None]
                assert np.array_equal(t.numpy(), got), f"step {i} {w}"
            ref = P.attend(rows[:, :b.Hq], c, o["row_start"], o["lens"], o["table"])
            tol, ltol = I.tolerance(dtype, np.nan_to_num(ref[0]), ref[1], np.nan_to_num(ref[2]), np.nan_to_num(ref[4]),
                                    b.most, D, c.value_size())
            a = b.a.numpy().astype(np.float64)
            assert (np.abs(a[live] - ref[0][live]) <= tol[live]).all(), f"step {i}"
            assert (np.abs(b.lse.numpy()[live] - ref[1][live]) <= ltol[live]).all(), f"step {i}"
            ca, sa = I.quantize(b.a.numpy().astype(np.float32).reshape(tokens, -1))
            y = _narrow(tn, I.linear(ca, sa, *I.quantize(b.w["o"])), dtype)
            got = b.y.numpy() if dtype == "float32" else b.y.bits()
            assert np.array_equal(got[live], y[live]), f"step {i}"
            yield got[live], b.lse.bits()[live]
    if graph is not None:
        L.check(lib.tn_graph_destroy(graph))


STEPS = [[40, 3, 0, 0], [1, 1, 17, 0], [1, 1, 1, 50], [1, -1, 1, 1], [1, 30, 1, 1], [-1, 1, 1, 1], [60, 1, -1, 1],
         [1, 1, 5, 1], [90, 90, 1, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_block_served_eager_and_captured(tn, dtype):
    eager = list(_loop(tn, dtype, STEPS, False))
    graph = list(_loop(tn, dtype, STEPS, True))
    for i, (a, b) in enumerate(zip(eager, graph)):
        assert all(x.tobytes() == y.tobytes() for x, y in zip(a, b)), f"step {i}"


# --- what later tokens hold costs a row nothing -----------------------------------------------


def _own_most(c):
    """For each row the largest size that a value of its own keys can have, [rows, 1, 1]."""
    most = np.zeros(int(c.row_start[-1]))
    for r, x in enumerate(c.lens):
        for i in range(c.rows[r]):
            t = np.arange(x - c.rows[r] + i + 1)
            at = np.unique((c.table[r, t // c.S] * c.S + t % c.S) // 16)
            most[c.row_start[r] + i] = 127.0 * float(np.max(c.cache.scale["v"][at], initial=0))
    return most[:, None, None]


@pytest.mark.parametrize("dtype, climb", [("float32", 12), ("bfloat16", 12), ("float16", 3)])
@pytest.mark.parametrize("H, G, D, rows, lens", [(2, 1, 64, [200], [200]), (1, 4, 128, [70, 1, 33], [300, 90, 40]),
                                                 (1, 2, 256, [100], [100]), (2, 3, 32, [150, 5], [150, 64])])
@MANY
def test_scales_of_later_tokens_cost_a_row_nothing(tn, many, dtype, climb, H, G, D, rows, lens):
    """Each block's values are 2^climb times the block's before it, over and over through eight blocks: a row in the
    middle of a tile is held to the bound of the keys that it attends."""
    c = Case(tn, dtype, H, G, D, 16, rows, lens, seed=21)
    for r, x in enumerate(lens):
        for b in range(-(-x // 16)):
            c.cache.scale["v"][c.table[r, b]] *= np.float32(2.0 ** (climb * (b % 8) - 4 * climb))
    out, lse = c.run(tn, many=many)
    ro, rl, pav, _, qk, _ = P.attend(c.q.numpy().astype(np.float64), c.cache, c.row_start, c.lens, c.table, None)
    tol, ltol = I.tolerance(dtype, ro, rl, pav, qk, max(lens), D, _own_most(c))
    worst, lworst = np.max(np.abs(out - ro) / tol), np.max(np.abs(lse - rl) / ltol)
    print(f"  worst {worst:.3f} of the bound, lse {lworst:.3f}", flush=True)
    assert worst <= 1 and lworst <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@MANY
def test_a_rows_bits_do_not_depend_on_later_tokens_values(tn, many, dtype):
    """The same rows with the values of a later block 2^40 and 2^-40 times as large."""
    c = Case(tn, dtype, 1, 2, 64, 16, [120], [120], seed=22)
    was, last = c.cache.scale["v"].copy(), c.table[0, 3]  # tokens 48 .. 63, in the same tile as all before
    got = []
    for mul in (1.0, 2.0 ** 40, 2.0 ** -40):
        c.cache.scale["v"][:] = was
        c.cache.scale["v"][last] *= np.float32(mul)
        got.append(c.run(tn, bits=True, many=many))
    for out, lse in got[1:]:
        assert np.array_equal(out[:48], got[0][0][:48]) and np.array_equal(lse[:48], got[0][1][:48])


# --- threads ------------------------------------------------------------------------------------


def test_threads_on_one_stream_share_layers_and_caches(tn):
    """Each thread's products and attention are its own, bit for bit, where all go through the same scratch."""
    import threading

    rng = np.random.default_rng(31)
    layer = tn.Int8Linear(tn.i8_quantize(_up(tn, rng.standard_normal((900, 700)).astype(np.float32))))
    c = Case(tn, "bfloat16", 2, 4, 128, 16, [1, 1, 1], [900, 1300, 40])
    dev, table = _fill(tn, c.cache), object.__new__(tn.PageTable)
    table.requests, table.width, table.page_size = 3, c.table.shape[1], c.S
    table.row_start, table.lens, table.table = (_ints(tn, a) for a in (c.row_start, c.lens, c.table))
    xs = [_up(tn, rng.standard_normal((70, 700)).astype(np.float32)) for _ in range(4)]
    qs = [_up(tn, rng.standard_normal((3, 8, 128)).astype(np.float32), "bfloat16") for _ in range(4)]
    want = [(layer(x).numpy(), dev.attend(q, table, 1, 1300)[0].bits()) for x, q in zip(xs, qs)]
    bad, go = [], threading.Barrier(4)

    def work(i):
        try:
            go.wait()
            for n in range(40):
                y, (a, _) = layer(xs[i]), dev.attend(qs[i], table, 1, 1300)
                if n % 8 == 7 and not (np.array_equal(y.numpy(), want[i][0]) and np.array_equal(a.bits(), want[i][1])):
                    bad.append((i, n))
        except Exception as e:  # noqa: BLE001
            bad.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert bad == []


# --- the digits of a probability ---------------------------------------------------------------


@pytest.mark.parametrize("H, G, D, rows, lens", [(2, 4, 64, [1, 1], [700, 300]), (1, 4, 128, [160, 3], [400, 90]),
                                                 (1, 2, 256, [90], [300])])
@MANY
def test_f16_rows_are_off_by_no_more_than_their_rounding(tn, many, H, G, D, rows, lens):
    """Probabilities are held in two f16 parts: the bound of f32 rows, and a half step of f16 for the output's rounding.
    In one part each is off by up to another half step, which some of these thousands of elements would show: queries of
    one element keep the scores' share of the bound small."""
    h = 2.0 ** -11
    c = Case(tn, "float16", H, G, D, 16, rows, lens, seed=23)
    x = 3 * c.q.numpy().astype(np.float32)
    x[..., 1:] = 0
    c.q = _up(tn, x, "float16")
    out, lse = c.run(tn, many=many)
    ro, rl, pav, _, qk, _ = P.attend(c.q.numpy().astype(np.float64), c.cache, c.row_start, c.lens, c.table, None)
    tol, ltol = I.tolerance("float32", ro, rl, pav, qk, max(lens), D, c.cache.value_size())
    tol = tol + h * (np.abs(ro) + tol) + 2.0 ** -25
    worst, lworst = np.max(np.abs(out - ro) / tol), np.max(np.abs(lse - rl) / ltol)
    off = float(np.linalg.norm(out - ro) / np.linalg.norm(ro))
    print(f"  worst {worst:.3f} of the bound, lse {lworst:.3f}, off by {off:.2e} of the norm", flush=True)
    assert worst <= 1 and lworst <= 1


# --- every shape of the product -----------------------------------------------------------------


@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_every_product_bit_for_bit(tn, m, n, k):
    """Quantised on the device and by the oracle; the sums of codes are whole numbers below 2^53, exact in f64."""
    rng = np.random.default_rng(m + n + k)
    odt = DTYPES[(m + n) % 3]
    x = rng.standard_normal((m, k)).astype(np.float32) * (0.5 + rng.random((m, 1))).astype(np.float32)
    w = rng.standard_normal((n, k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    tx, tw = _up(tn, x, DTYPES[m % 3]), tn.i8_quantize(_up(tn, w))
    cx, sx = I.quantize(tx.numpy().astype(np.float32))
    cw, sw = I.quantize(w)
    print(f"case [{m}, {k}] x [{n}, {k}] {tx.dtype} -> {odt}", flush=True)
    total = (cx.astype(np.float64) @ cw.T.astype(np.float64)).astype(np.float32)
    want = _narrow(tn, ((total * sw[None]).astype(np.float32) * sx[:, None]).astype(np.float32) + b, odt)
    got = tn.i8_linear(tx, tw, _up(tn, b), out_dtype=odt)
    got = got.numpy() if odt == "float32" else got.bits()
    assert got.tobytes() == want.tobytes(), np.argwhere(got != want)[:5]
    a = tn.i8_quantize(tx)
    assert np.array_equal(a.codes.numpy()[:, :k], cx)
    again = tn.i8_matmul(a, tw, _up(tn, b), out_dtype=odt)
    assert (again.numpy() if odt == "float32" else again.bits()).tobytes() == want.tobytes()
