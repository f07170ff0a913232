"""The loss head without logits and Muon as a user has them: through the C++ API
(tests/native/loss_and_muon_check.cpp) and in the trainer's step, together and each alone."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import veda_b200 as V
from oracle import veda_oracle as O

ROOT = Path(__file__).resolve().parent.parent
ADAM = O.AdamWConfig(1e-3, 0.9, 0.95, 1e-8, 0.1)
QWEN = O.ModelConfig(vocab=2048, hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, head_dim=128, eps=1e-6,
                     theta=1e6)
NS = (3.4445, -4.7750, 2.0315)


def trainer(cfg, dtype, batch, seq_len, params):
    from veda_b200.train_abi import Trainer
    t = Trainer(cfg, lr=ADAM.learning_rate, betas=(ADAM.beta1, ADAM.beta2), eps=ADAM.eps,
                weight_decay=ADAM.weight_decay, max_norm=1.0, dtype=dtype, batch=batch, seq_len=seq_len, seed=0)
    t.set_params(np.concatenate([p.ravel() for p in params]))
    return t


def split(cfg, flat):
    out, at = [], 0
    for _, shape in O.param_specs(cfg):
        n = int(np.prod(shape))
        out.append(flat[at:at + n].reshape(shape))
        at += n
    return out


def compile_check(tmp):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp / "loss_and_muon_check"
    subprocess.run([cxx, "-std=c++23", "-O1", "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "native" / "loss_and_muon_check.cpp"), "-o", str(exe), "-L",
                    str(V.PKG), "-lveda", "-lveda_cuda", f"-Wl,-rpath,{V.PKG}"], check=True)
    return exe


def test_cpp_api_compiles(tmp_path):
    compile_check(tmp_path)


@pytest.mark.gpu
def test_cpp_api(cuda, tmp_path):
    r = subprocess.run([str(compile_check(tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("cfg,dtype,B,T,tol", [(O.TINY, 0, 4, 32, 1e-4), (QWEN, 1, 2, 128, 2e-2)])
def test_step_with_the_linear_loss_against_the_oracle(cuda, cfg, dtype, B, T, tol):
    params = O.init_params(cfg, 3, bf16=dtype == 1)
    ids, tg = O.synthetic_batch(cfg, B, T, 3)
    t = trainer(cfg, dtype, B, T, params)
    t.set_linear_loss(True)
    loss, norm = t.step_host(ids, tg)
    got = split(cfg, t.get_grads())
    t.close()
    ref = [p.copy() for p in params]
    rloss, rnorm, rgrads = O.train_step(cfg, ref, ids, tg, 1.0, O.AdamW(ref, ADAM))
    assert abs(loss - rloss) <= tol * abs(rloss) and abs(norm - rnorm) <= tol * rnorm
    assert max(O.max_abs_rel(a, b) for a, b in zip(got, rgrads)) <= tol


@pytest.mark.gpu
def test_linear_loss_does_not_count_ignored_targets(cuda):
    # a batch whose second sequence is padding has the gradients of the first alone: the embedding
    # scatter sees zero rows for it
    params = O.init_params(QWEN, 4, bf16=True)
    ids, tg = O.synthetic_batch(QWEN, 2, 128, 4)
    two = trainer(QWEN, 1, 2, 128, params)
    two.set_linear_loss(True)
    one = trainer(QWEN, 1, 1, 128, params)
    one.set_linear_loss(True)
    pad = tg.copy().reshape(2, 128)
    pad[1] = -100
    l2, _ = two.step_host(ids, pad.reshape(tg.shape))
    l1, _ = one.step_host(ids.reshape(2, 128)[:1], tg.reshape(2, 128)[:1])
    a, b = split(QWEN, two.get_grads()), split(QWEN, one.get_grads())
    two.close()
    one.close()
    assert l1 == l2
    # the same rows through products of other sizes: bf16 roundings of the activations' gradients
    assert max(O.max_abs_rel(x, y) for x, y in zip(a, b)) <= 2e-2


def orthogonalized(u, steps=5, eps=1e-7):
    x = u.astype(np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.linalg.norm(x) + eps)
    for _ in range(steps):
        s = x @ x.T
        x = NS[0] * x + (NS[1] * s + NS[2] * s @ s) @ x
    return x.T if tall else x


def is_hidden(name, shape):
    return len(shape) == 2 and "embed" not in name


@pytest.mark.gpu
@pytest.mark.parametrize("cfg,dtype,B,T", [(O.TINY, 0, 4, 32), (QWEN, 1, 2, 128)])
@pytest.mark.parametrize("linear", [False, True])
def test_muon_steps_in_the_trainer(cuda, cfg, dtype, B, T, linear):
    params = O.init_params(cfg, 5, bf16=dtype == 1)
    ids, tg = O.synthetic_batch(cfg, B, T, 5)
    t = trainer(cfg, dtype, B, T, params)
    t.set_linear_loss(linear)
    lr, mom, wd = 2e-3, 0.95, 0.1
    t.use_muon(lr, mom, True, wd)
    w = [p.astype(np.float64) for p in params]
    m = [np.zeros_like(p) for p in w]
    plain = trainer(cfg, dtype, B, T, params)   # AdamW alone: what the other parameters do
    plain.set_linear_loss(linear)
    for k in range(3):
        loss, norm = t.step_host(ids, tg)
        grads = split(cfg, t.get_grads())
        got = split(cfg, t.get_params())
        clip = 1.0 / norm if norm > 1.0 else 1.0
        for i, (name, shape) in enumerate(O.param_specs(cfg)):
            if not is_hidden(name, shape):
                w[i] = got[i].astype(np.float64)
                continue
            g = grads[i].astype(np.float64) * clip
            m[i] = mom * m[i] + g
            step = lr * 0.2 * max(shape) ** 0.5
            w[i] = w[i] * (1 - lr * wd) - step * orthogonalized(g + mom * m[i])
            # the update is within 0.3 % of its size (fp16 products; fp32: far less), the weights are
            # rounded to fp32; over the steps taken
            tol = (k + 1) * (3e-3 * step * min(shape) ** 0.5 + 4 * 2.0 ** -24 * np.linalg.norm(w[i]))
            assert np.linalg.norm(got[i] - w[i]) <= tol, (k, name, np.linalg.norm(got[i] - w[i]) / tol)
        if k == 0:
            plain.step_host(ids, tg)
            other = split(cfg, plain.get_params())
            for i, (name, shape) in enumerate(O.param_specs(cfg)):
                if not is_hidden(name, shape):
                    assert np.array_equal(got[i], other[i]), name
    t.close()
    plain.close()


@pytest.mark.gpu
@pytest.mark.parametrize("cfg,dtype,B,T", [(O.TINY, 0, 4, 32), (QWEN, 1, 2, 128)])
def test_graph_replay_checkpoint_and_eager_agree_bit_for_bit(cuda, cfg, dtype, B, T, tmp_path):
    params = O.init_params(cfg, 6, bf16=dtype == 1)
    batches = [O.synthetic_batch(cfg, B, T, 10 + k) for k in range(5)]

    def run(graph, resume=False):
        t = trainer(cfg, dtype, B, T, params)
        t.set_step_graph(graph)
        t.set_linear_loss(True)
        t.use_muon(1e-3)
        out = []
        for k, (ids, tg) in enumerate(batches):
            if resume and k == 3:
                t.save(str(tmp_path / f"c{dtype}"))
                t.close()
                t = trainer(cfg, dtype, B, T, params)
                t.set_step_graph(graph)
                t.set_linear_loss(True)
                t.use_muon(1e-3)
                t.load(str(tmp_path / f"c{dtype}"))
            out.append(t.step_host(ids, tg))
        w = t.get_params()
        t.close()
        return out, w

    eager, replay, resumed = run(False), run(True), run(True, resume=True)
    assert eager[0] == replay[0] == resumed[0]
    assert np.array_equal(eager[1], replay[1]) and np.array_equal(eager[1], resumed[1])


@pytest.mark.gpu
def test_switching_while_training(cuda):
    # logits -> linear loss -> logits, AdamW -> Muon -> Muon with other numbers: each step runs, and a
    # refused configuration leaves the one before in place
    cfg, B, T = O.TINY, 4, 32
    params = O.init_params(cfg, 7)
    ids, tg = O.synthetic_batch(cfg, B, T, 7)
    t = trainer(cfg, 0, B, T, params)
    losses = []
    for k in range(8):
        if k == 2:
            t.set_linear_loss(True)
        if k == 4:
            t.use_muon(1e-3)
            with pytest.raises((ValueError, RuntimeError), match="momentum"):
                t.use_muon(1e-3, momentum=1.5)
            with pytest.raises((ValueError, RuntimeError), match="step"):
                t.use_muon(1e-3, steps=0)
        if k == 6:
            t.set_linear_loss(False)
            t.use_muon(2e-3, nesterov=False)
        losses.append(t.step_host(ids, tg)[0])
    t.close()
    assert np.isfinite(losses).all()


@pytest.mark.gpu
def test_skipped_step_leaves_muon_alone(cuda):
    cfg, B, T = O.TINY, 4, 32
    params = O.init_params(cfg, 8)
    ids, tg = O.synthetic_batch(cfg, B, T, 8)
    t = trainer(cfg, 0, B, T, params)
    t.use_muon(1e-3)
    t.set_skip_nonfinite(True)
    w = t.get_params()
    bad = w.copy()
    at = sum(int(np.prod(s)) for _, s in O.param_specs(cfg)) - 1
    bad[at] = np.inf   # an infinite gain in the final norm
    t.set_params(bad)
    t.step_host(ids, tg)
    assert t.step_skipped() and np.array_equal(t.get_params(), bad)
    t.set_params(w)
    loss, norm = t.step_host(ids, tg)
    assert not t.step_skipped() and np.isfinite(loss) and np.isfinite(norm) and np.isfinite(t.get_params()).all()
    t.close()
