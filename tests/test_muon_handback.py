"""What AdamW makes of parameters that Muon had: given back in the C++ API (tests/native/muon_handback_check.cpp), and
loaded from the checkpoint of a trainer with Muon."""
import json
import shutil
import struct
import subprocess
from pathlib import Path

import numpy as np
import pytest

import veda_b200 as V
from oracle import veda_oracle as O
from tests.test_loss_and_muon_step import ADAM, QWEN, is_hidden, split, trainer

ROOT = Path(__file__).resolve().parent.parent


def compile_check(tmp):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp / "muon_handback_check"
    subprocess.run([cxx, "-std=c++23", "-O1", "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "native" / "muon_handback_check.cpp"), "-o", str(exe), "-L", str(V.PKG), "-lveda",
                    "-lveda_cuda", f"-Wl,-rpath,{V.PKG}"], check=True)
    return exe


def test_compiles(tmp_path):
    compile_check(tmp_path)


@pytest.mark.gpu
def test_cpp_api(cuda, tmp_path):
    r = subprocess.run([str(compile_check(tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr


def metadata(directory):
    raw = (Path(directory) / "optimizer.safetensors").read_bytes()
    (n,) = struct.unpack("<Q", raw[:8])
    return json.loads(raw[8:8 + n])["__metadata__"]


@pytest.mark.gpu
@pytest.mark.parametrize("cfg,dtype,B,T", [(O.TINY, 0, 4, 32), (QWEN, 1, 2, 128)])
@pytest.mark.parametrize("graph", [False, True])
def test_checkpoint_of_muon_in_a_trainer_without_it(cuda, cfg, dtype, B, T, graph, tmp_path):
    params = O.init_params(cfg, 9, bf16=dtype == 1)
    batches = [O.synthetic_batch(cfg, B, T, 20 + k) for k in range(16)]
    t = trainer(cfg, dtype, B, T, params)
    t.use_muon(1e-3)
    for k in range(8):
        t.step_host(*batches[k])
    t.save(str(tmp_path / "a"))
    t.close()
    hidden = [name for name, shape in O.param_specs(cfg) if is_hidden(name, shape)]
    assert sorted(metadata(tmp_path / "a")["muon"].split(",")) == sorted(hidden)

    t = trainer(cfg, dtype, B, T, params)
    t.set_step_graph(graph)
    for k in range(3):
        t.step_host(*batches[k])   # a step graph is there when the checkpoint comes
    t.load(str(tmp_path / "a"))
    before = split(cfg, t.get_params())
    t.step_host(*batches[8])
    after = split(cfg, t.get_params())
    for (name, shape), p, q in zip(O.param_specs(cfg), before, after):
        if is_hidden(name, shape):
            # AdamW's first step: lr in size, beside the decay, and fp32's roundings of the weights
            off = np.abs(q.astype(np.float64) - p) - ADAM.learning_rate * (1 + ADAM.weight_decay * np.abs(p))
            assert (off <= 1e-4 * ADAM.learning_rate + 2.0 ** -22 * np.abs(p)).all(), (name, off.max() / ADAM.learning_rate)
    # the corrections' beginning is kept: a second resume goes on bit for bit
    t.step_host(*batches[9])
    t.save(str(tmp_path / "b"))
    assert "muon" not in metadata(tmp_path / "b")
    one = [t.step_host(*batches[k]) for k in range(10, 14)]
    w = t.get_params()
    t.close()
    t = trainer(cfg, dtype, B, T, params)
    t.set_step_graph(graph)
    t.load(str(tmp_path / "b"))
    two = [t.step_host(*batches[k]) for k in range(10, 14)]
    assert one == two and np.array_equal(w, t.get_params())
    # and from there to Muon, with AdamW's first moment as its momentum
    t.use_muon(1e-3)
    for k in range(14, 16):
        loss, norm = t.step_host(*batches[k])
    assert np.isfinite(loss) and np.isfinite(norm) and np.isfinite(t.get_params()).all()
    t.close()


@pytest.mark.gpu
def test_muon_with_other_numbers_keeps_its_momentum(cuda):
    cfg, B, T = O.TINY, 4, 32
    params = O.init_params(cfg, 10)
    ids, tg = O.synthetic_batch(cfg, B, T, 10)
    a, b = (trainer(cfg, 0, B, T, params) for _ in range(2))
    for t in (a, b):
        t.use_muon(1e-3)
        for _ in range(3):
            t.step_host(ids, tg)
    b.use_muon(1e-3)   # the same numbers again
    assert a.step_host(ids, tg) == b.step_host(ids, tg) and np.array_equal(a.get_params(), b.get_params())
    a.close()
    b.close()


@pytest.mark.gpu
def test_profile_class_of_muon(cuda):
    from veda_b200 import train_abi as TA
    cfg, B, T = QWEN, 2, 128
    params = O.init_params(cfg, 11, bf16=True)
    ids, tg = O.synthetic_batch(cfg, B, T, 11)
    t = trainer(cfg, 1, B, T, params)
    t.use_muon(1e-3)
    t.step_host(ids, tg)
    TA.profile_enable(True)
    try:
        t.step_host(ids, tg)
        got = TA.profile_collect()
    finally:
        TA.profile_enable(False)
    t.close()
    shapes = [shape for name, shape in O.param_specs(cfg) if is_hidden(name, shape)]
    taken = sum(int(np.prod(s)) for s in shapes)
    every = sum(int(np.prod(s)) for _, s in O.param_specs(cfg))
    flops = sum(5.0 * (m * m * n + m ** 3 + 2.0 * m * m * n) for m, n in ((min(s), max(s)) for s in shapes))
    ms, f, b, n = got["muon"]
    assert n == 1 and ms > 0 and b == 22.0 * taken and abs(f - flops) <= 1e-9 * flops
    ms, f, b, n = got["adamw"]
    # every gradient for the norm; gradient, moments and masters of the rest
    assert n == 1 and ms > 0 and b == 4.0 * every + 30.0 * (every - taken)
