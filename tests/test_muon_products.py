"""optim::MuonConfig::fp32_products through the C++ API (tests/native/muon_products_check.cpp)."""
import subprocess

import pytest

from tests.test_loss_views import compile_check


def test_compiles(tmp_path):
    compile_check("muon_products_check", tmp_path)


@pytest.mark.gpu
def test_cpp_api(cuda, tmp_path):
    r = subprocess.run([str(compile_check("muon_products_check", tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr
