"""A cluster query that fails is asked again at the next call (host code against a fake of the failing call)."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import ctypes, sys
import veda_b200 as V
lib, fake = V.lib(), ctypes.CDLL(sys.argv[1])
A = 1 << 20   # never read
def orth(dtype):
    return lib.veda_orthogonalize(A, 304, 304 * 304, A, 304, 304 * 304, 1, 304, 304, 5, 3.4445, -4.7750, 2.0315, 1e-7,
                                  A, 1 << 40, dtype, None)
def muon(lowp):
    return lib.veda_muon_step(A, A, A, lowp, 1, 304, 304, 304 * 304, 1e-3, 0.9, 1, 0.1, 1.0, 5, 3.4445, -4.7750, 2.0315,
                              1e-7, None, 1.0, 1.0, 0, A, 1 << 40, None)
def fwd(dtype):
    return lib.veda_linear_cross_entropy_fwd(A, 64, A, 64, A, -100, A, A, A, 304, 5000, 64, A, 1 << 40, None, dtype, None)
def bwd(dtype):
    return lib.veda_linear_cross_entropy_bwd(A, 64, A, 64, A, -100, A, None, A, 64, A, 64, V.F32, 0.0, 304, 5000, 64, A,
                                             1 << 40, None, dtype, None)
for call, arg in ((orth, V.BF16), (orth, V.F32), (muon, A), (muon, None), (fwd, V.BF16), (fwd, V.F32), (bwd, V.BF16),
                  (bwd, V.F32)):
    fake.fake_fail_queries(1)
    rc = call(arg)
    assert rc == V.ERR_CUDA, (call.__name__, arg, rc, lib.veda_last_error())
    assert b"query" in lib.veda_last_error(), lib.veda_last_error()
    for _ in range(2):
        before = fake.fake_launches()
        assert call(arg) == V.OK, (call.__name__, arg, lib.veda_last_error())
        assert fake.fake_launches() > before
print("ok")
"""


def test_a_failed_cluster_query_is_asked_again(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    fake = tmp_path / "fake_cudart.so"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", str(ROOT / "tests" / "native" / "fake_cudart.cpp"), "-o",
                    str(fake)], check=True)
    r = subprocess.run([sys.executable, "-c", SCRIPT, str(fake)], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env={**os.environ, "LD_PRELOAD": str(fake)})
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
