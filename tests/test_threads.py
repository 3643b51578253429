"""Several threads on one stream: the launches of a call that share a buffer, the caller's or the library's, follow one
another with no other call's between them. And scratch that ends with its stream. Run over tests/hip_record.cpp, which records launches and runs none."""

import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = r"""
import ctypes, sys, threading, time
R = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # ahead of the library's own runtime
from torchnative_amd import _lib
L = _lib.lib()
NAN = float("nan")
P = 1 << 20                      # a pointer that nothing follows
HOST = (ctypes.c_int64 * 4)(0, 0, 0, 0)
q4 = _lib.Q4Cache(P, P, P, P, 4096, 16, 8, 128)
q8 = _lib.Q8Cache(P, P, P, P, 4096, 16, 8, 128)
big = 1 << 40


def paged(fn, cache, n, tokens, rows, most):
    return lambda st: fn(st, ctypes.byref(cache), 1, P, 32 * 128, tokens, 32, n, P, P, P, 4096, rows, most, NAN, P, big,
                         P, P)


def llama():
    layer = _lib.LlamaLayer()
    for f, _ in _lib.LlamaLayer._fields_:
        setattr(layer, f, _lib.Q4Weight(P, P) if f in ("qkv", "o", "gate_up", "down") else P)
    layers = (_lib.LlamaLayer * 1)(layer)
    m = _lib.Llama()
    for f, t in _lib.Llama._fields_:
        if t is ctypes.c_void_p:
            setattr(m, f, P)
        elif t is _lib.Q4Weight:
            setattr(m, f, _lib.Q4Weight(P, P))
    m.layers = ctypes.cast(layers, type(m.layers)) if hasattr(m, "layers") else None
    m.n_layers, m.hidden, m.n_heads, m.n_kv_heads, m.head_dim, m.inter, m.vocab = 1, 576, 9, 3, 64, 1536, 4096
    m.cap, m.prompt_len = 256, 64
    for f in ("eps", "norm_eps"):
        if hasattr(m, f):
            setattr(m, f, 1e-5)
    m._keep = layers
    return m


model = llama()
CALLS = {
    "i8_linear": lambda st: L.tn_i8_linear(st, P, 1, 64, 4096, P, P, 4096, None, P, big, big, 1),
    "sdpa_paged_q8 few": paged(L.tn_sdpa_paged_q8, q8, 16, 16, 1, 4096),
    "sdpa_paged_q8 many": paged(L.tn_sdpa_paged_q8, q8, 1, 512, 512, 20000),
    "sdpa_paged_q4_0 few": paged(L.tn_sdpa_paged_q4_0, q4, 16, 16, 1, 4096),
    "sdpa_paged_q4_0 many": paged(L.tn_sdpa_paged_q4_0, q4, 1, 512, 512, 20000),
    "q4_0_linear": lambda st: L.tn_q4_0_linear(st, P, 0, 64, 4096, P, P, 4096, None, P, 0),
    "q8_0_linear": lambda st: L.tn_q8_0_linear(st, P, 0, 64, 4096, P, P, 4096, None, P, 0),
    "q4_k_linear": lambda st: L.tn_q4_k_linear(st, P, 0, 64, 4096, P, 4096, None, P, 0),
    "sdpa_fwd": lambda st: L.tn_sdpa_fwd(st, 1, P, P, P, 1, 4, 1, 300, 4096, 96, None, 0, None, 0, NAN, P, P),
    "sdpa_decode": lambda st: L.tn_sdpa_decode(st, 0, P, P, P, 2, 9, 3, 4096, 64, P, 4096, NAN, P, P),
    "sdpa_decode_noalloc": lambda st: L.tn_sdpa_decode_noalloc(st, 0, P, P, P, 2, 9, 3, 4096, 64, P, 4096, NAN, P, P),
    "llama_step": lambda st: L.tn_llama_step(st, ctypes.byref(model)),
    "llama_prefill": lambda st: L.tn_llama_prefill(st, ctypes.byref(model), 64, P),
}


def log():
    n = R.record_launches(None, 0)
    out = (ctypes.c_int64 * (2 * max(n, 1)))()
    R.record_launches(out, n)
    return [out[2 * i] for i in range(n)]


name = sys.argv[2]
call = CALLS[name]
stream = ctypes.c_void_p()
_lib.check(L.tn_stream_create(ctypes.byref(stream)))
for st in (None, stream.value):
    _lib.check(call(st))  # (workspaces grow here)
    R.record_clear()
    _lib.check(call(st))
    k = len(log())
    assert k > 1, f"{name}: {k} launch"
    R.record_clear()
    go = threading.Barrier(3)

    def work(i):
        R.record_thread(i)
        go.wait()
        for _ in range(30):
            _lib.check(call(st))
            time.sleep(2e-4)

    threads = [threading.Thread(target=work, args=(i,)) for i in (1, 2, 3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    seen = log()
    assert len(seen) == 90 * k
    parts = [set(seen[i:i + k]) for i in range(0, len(seen), k)]
    mixed = sum(len(p) > 1 for p in parts)
    print(f"{name}: {k} launches a call, {mixed} of {len(parts)} calls had another's among theirs")
    assert mixed == 0
    assert sum(a != b for a, b in zip(parts, parts[1:])) > 2, "the threads did not take turns: nothing was tested"
"""

NAMES = ["i8_linear", "sdpa_paged_q8 few", "sdpa_paged_q8 many", "sdpa_paged_q4_0 few", "sdpa_paged_q4_0 many",
         "q4_0_linear", "q8_0_linear", "q4_k_linear", "sdpa_fwd", "sdpa_decode", "sdpa_decode_noalloc", "llama_step",
         "llama_prefill"]


@pytest.mark.parametrize("name", NAMES)
def test_launches_of_a_call_stay_together(recorder, name):
    r = subprocess.run([sys.executable, "-c", CHILD, recorder, name], capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(HERE))
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]


ENDS = r"""
import ctypes, gc, sys
R = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import torchnative_amd as tn
from torchnative_amd import _C
T = sys.modules["torchnative_amd.tensor"]


def events():
    n = R.record_events(None, 0)
    out = (ctypes.c_int64 * (2 * max(n, 1)))()
    R.record_events(out, n)
    return [(out[2 * i], out[2 * i + 1]) for i in range(n)]


GIVEN, FREED, WAITED, ENDED = 1, 2, 3, 4
x, w, y = tn.empty((64, 256)), tn.I8Rows((128, 256)), tn.empty((64, 128))
cache, table = tn.Q8Cache(512, 16, 8, 128), object.__new__(tn.PageTable)
table.requests, table.width, table.page_size = 1, 512, 16
table.row_start, table.lens, table.table = (tn.empty((n,), "int32") for n in (2, 1, 512))
q, out, lse = tn.empty((1, 32, 128)), tn.empty((1, 32, 128)), tn.empty((1, 32))


def calls():
    tn.i8_linear(x, w, out=y)
    cache.attend(q, table, 1, 8000, out=out, lse=lse)


calls()
always = _C._i8_work._held[0, None] + cache._work._held[0, None]  # the default stream's
for rnd in range(3):
    s = tn.Stream()
    R.record_clear()
    with s:
        calls()
        tn.i8_linear(tn.empty((640, 256)), w, out=tn.empty((640, 128)))  # outgrows the first
    handle = s.handle
    held = [t.data_ptr() for o in (_C._i8_work, cache._work) for t in o._held[0, handle]]
    assert len(held) == 3, held
    was = events()
    assert all((GIVEN, p) in was and (FREED, p) not in was for p in held), "another stream's buffer"
    R.record_clear()
    del s
    gc.collect()
    seen = events()
    print(seen)
    end = seen.index((ENDED, handle))
    for p in held:
        assert (FREED, p) in seen, "a buffer outlives its stream"
        assert seen.index((WAITED, handle)) < seen.index((FREED, p)) and seen.index((WAITED, handle)) < end
    assert list(_C._i8_work._held) == [(0, None)] and list(cache._work._held) == [(0, None)]
assert _C._i8_work._held[0, None] + cache._work._held[0, None] == always
"""


def test_scratch_ends_with_its_stream(recorder):
    """Its buffers are free for others only when its work has ended, and none stays behind."""
    r = subprocess.run([sys.executable, "-c", ENDS, recorder], capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(HERE))
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]
