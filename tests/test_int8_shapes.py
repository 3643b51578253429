"""Sizes that reach every shape of the int8 product, for the comparison with the oracle on the GPU: which kernel a size
gets is asked of the library itself, over tests/hip_record.cpp, so that a table that is tuned anew cannot leave one of its
shapes untested."""

import json
import os
import subprocess
import sys

# (m, n, k): odd rows and channels, k off a stage's 128 bytes
PRODUCTS = [
    (3, 70, 130), (16, 300, 1000),
    (33, 700, 100), (121, 113, 309), (300, 701, 640),  # 64 x 32
    (951, 589, 146), (39, 8337, 33),  # 64 x 64, two groups
    (241, 4991, 111),  # 64 x 64
    (1025, 1000, 1000), (527, 2417, 1171), (67, 12917, 986),  # 64 x 128, two groups
    (777, 5000, 128), (156, 15527, 157),  # 64 x 128
    (700, 8200, 320), (131, 27583, 193), (714, 10411, 183),  # 128 x 128
    (513, 20000, 128), (2042, 6657, 101),  # 256 x 256, whole tiles
    (1801, 3590, 7000), (1999, 4001, 6401),  # halved ones, the last with rows in its first half alone, and in both
    (2040, 12285, 810),  # both in one call
]

CHILD = r"""
import ctypes, json, sys
R = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # ahead of the library's own runtime
R.record_kernel.restype = R.record_registered.restype = ctypes.c_char_p
from torchnative_amd import _lib
L, P, out = _lib.lib(), 1 << 20, []
for m, n, k in json.loads(sys.argv[2]):
    R.record_clear()
    _lib.check(L.tn_i8_linear(None, P, 0, m, k, P, P, n, None, P, 1 << 50, 1 << 50, 0))
    last = R.record_launches(None, 0) - 1
    out.append((R.record_kernel(last).decode(), R.record_workgroups(last)))
names, i = [], 0
while R.record_registered(i):
    names.append(R.record_registered(i).decode())
    i += 1
print(json.dumps([out, names]))
"""


def test_every_product_is_reached(recorder):
    r = subprocess.run([sys.executable, "-c", CHILD, recorder, json.dumps(PRODUCTS)], capture_output=True, text=True,
                       timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]
    got, names = json.loads(r.stdout)
    for what, count in (("k_i8_gemm", 6), ("k_i8_large", 1), ("k_i8_few", 1), ("k_i8_fused", 3)):
        kernels = {n for n in names if what in n}
        assert len(kernels) == count, kernels
        missing = kernels - {k for k, _ in got}
        # (one of k_i8_fused's three types: the others differ in how they load a row)
        assert not missing or what == "k_i8_fused" and len(missing) == 2, missing
    kinds = set()
    for (m, n, _), (kernel, workgroups) in zip(PRODUCTS, got):
        if "k_i8_large" in kernel:
            tiles = -(-m // 256) * -(-n // 256)
            halved = workgroups - tiles
            assert 0 <= halved <= tiles
            kinds.add((halved > 0, halved < tiles))
    assert kinds == {(False, True), (True, False), (True, True)}, kinds


BESIDE = r"""
import ctypes, sys
R = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from torchnative_amd import _lib
L = _lib.lib()
m, n, k, x, w, far = 3, 100, 200, 1 << 20, 1 << 24, 1 << 28
for y in (x + m * k * 2, x - m * n * 4, w + n * 256, w - m * n * 4):
    _lib.check(L.tn_i8_linear(None, x, 1, m, k, w, far, n, None, None, 0, y, 0))
for y in (x + m * 256, x - m * n * 4, w + n * 256):
    _lib.check(L.tn_i8_matmul(None, x, far, m, k, w, far, n, None, y, 0))
assert R.record_launches(None, 0) == 7
"""


def test_an_output_beside_its_inputs_is_taken(recorder):
    r = subprocess.run([sys.executable, "-c", BESIDE, recorder], capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]
