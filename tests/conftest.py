import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) and the built HIP library")


@pytest.fixture(scope="session")
def recorder(tmp_path_factory):
    """A HIP runtime that records launches and runs none (hip_record.cpp), for a process to load ahead of the library."""
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    out = str(tmp_path_factory.mktemp("hip") / "librecord.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-pthread", "-o", out,
                    os.path.join(ROOT, "tests", "hip_record.cpp")], check=True)
    return out


@pytest.fixture(scope="session")
def golden():
    import json

    with open(os.path.join(ROOT, "tests", "golden", "golden_gguf_py.json")) as fh:
        doc = json.load(fh)
    return {(c["format"], c["name"]): c for c in doc["cases"]}, doc
