"""How the CTA-pair kernels are launched (host code against a fake CUDA runtime): with SMs of their own, and never
overlapping a launch of another kind, beside whose last blocks their tensor memory would be allocated."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

import veda_b200 as V
from tests.gpu_util import call, empty, ptr, stream, sync, torch, workspace

ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import ctypes, sys
import veda_b200 as V
lib, fake = V.lib(), ctypes.CDLL(sys.argv[1])
A = 1 << 20   # never read
NS = (3.4445, -4.7750, 2.0315, 1e-7)
calls = []
for dtype in (V.BF16, V.F32):
    for base in (A, A + 4):   # read in place or laid out first
        for rows, vocab, dim in ((300, 5000, 64), (2048, 32000, 1024)):
            calls.append(lambda d=dtype, b=base, s=(rows, vocab, dim): lib.veda_linear_cross_entropy_fwd(
                b, s[2], b, s[2], A, -100, A, A, A, *s, A, 1 << 50, None, d, None))
            calls.append(lambda d=dtype, b=base, s=(rows, vocab, dim): lib.veda_linear_cross_entropy_bwd(
                b, s[2], b, s[2], A, -100, A, None, A, s[2], A, s[2], V.F32, 0.0, *s, A, 1 << 50, None, d, None))
    calls.append(lambda d=dtype: lib.veda_orthogonalize(A, 304, 304 * 304, A, 304, 304 * 304, 2, 304, 304, 5, *NS, A,
                                                        1 << 50, d, None))
one, pairs, overlapped = [ctypes.c_int() for _ in range(3)], 0, 0
for call in calls + calls[::-1]:
    first = fake.fake_launches()
    assert call() == V.OK, lib.veda_last_error()
    before = None
    for i in range(first, fake.fake_launches()):
        fake.fake_launch(i, *[ctypes.byref(v) for v in one])
        smem, over, coop = (v.value for v in one)
        if smem > 100 * 1024:
            assert smem == 227 * 1024, smem
            assert not over or (before is not None and before > 100 * 1024), (i - first, before)
            assert not (over and coop)
            pairs, overlapped = pairs + 1, overlapped + over
        before = smem
assert pairs > 30 and overlapped > 10, (pairs, overlapped)
print("ok")
"""


def test_pair_kernels_own_their_sms_and_overlap_only_one_another(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    fake = tmp_path / "fake_cudart.so"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", str(ROOT / "tests" / "native" / "fake_cudart.cpp"), "-o",
                    str(fake)], check=True)
    r = subprocess.run([sys.executable, "-c", SCRIPT, str(fake)], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env={**os.environ, "LD_PRELOAD": str(fake)})
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,vocab,dim", [(V.F32, 1100, 12000, 512), (V.BF16, 1100, 12000, 516)])
def test_many_calls_in_a_row_repeat_one(cuda, dtype, rows, vocab, dim):
    t = torch()
    g = t.Generator(device="cuda").manual_seed(31)
    dt = t.float32 if dtype == V.F32 else t.bfloat16
    x = t.randn(rows, dim, device="cuda", generator=g).to(dt)
    w = (t.randn(vocab, dim, device="cuda", generator=g) * 0.05).to(dt)
    tg = t.randint(0, vocab, (rows,), device="cuda", generator=g)
    ws = workspace(max(V.lib().veda_linear_cross_entropy_workspace(rows, vocab, dim, dim, dim, dtype, k) for k in (0, 1)))
    row, lse, loss, dx, dw = empty((rows,)), empty((rows,)), empty((1,)), empty((rows, dim), dtype), empty((vocab, dim), dtype)

    def step():
        call("veda_linear_cross_entropy_fwd", ptr(x), dim, ptr(w), dim, ptr(tg), -100, ptr(row), ptr(lse), ptr(loss), rows,
             vocab, dim, ptr(ws), ws.numel(), None, dtype, stream())
        call("veda_linear_cross_entropy_bwd", ptr(x), dim, ptr(w), dim, ptr(tg), -100, ptr(lse), None, ptr(dx), dim, ptr(dw),
             dim, dtype, 0.0, rows, vocab, dim, ptr(ws), ws.numel(), None, dtype, stream())

    step()
    want = [v.clone() for v in (row, lse, loss, dx, dw)]
    for _ in range(200):
        step()
    sync()
    assert all(bool((a == b).all()) for a, b in zip((row, lse, loss, dx, dw), want))
