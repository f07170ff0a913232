"""autograd::linear_cross_entropy on views and on a shared weight (tests/native/loss_views_check.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

import veda_b200 as V

ROOT = Path(__file__).resolve().parent.parent


def compile_check(name, tmp):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp / name
    subprocess.run([cxx, "-std=c++23", "-O1", "-I", str(ROOT / "include"), str(ROOT / "tests" / "native" / f"{name}.cpp"),
                    "-o", str(exe), "-L", str(V.PKG), "-lveda", "-lveda_cuda", f"-Wl,-rpath,{V.PKG}"], check=True)
    return exe


def test_compiles(tmp_path):
    compile_check("loss_views_check", tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("part", ["shared", "views"])
def test_cpp_api(cuda, tmp_path, part):
    r = subprocess.run([str(compile_check("loss_views_check", tmp_path)), part], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr
