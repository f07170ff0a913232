"""veda_orthogonalize and veda_muon_step against their formulas in 64 bits.

Tolerances, in the 2-norm over a matrix (the Frobenius norm), relative to the result. What the
kernels round is known: X to 22 bits as two fp16 values, S and P (and X in the products) to fp16 for
bf16 matrices, or to 22 bits for fp32 ones. `rounded()` runs the iteration in 64 bits with these
roundings alone; its distance from the exact result is the error that the choice of types costs on
that matrix. The kernels may add to it:
  * fp32 accumulation in the tensor cores: a sum of k terms, 16 to an instruction, is off by about
    2^-24 sqrt(k / 16 + 1) of its terms' size, three products an iteration, amplified by at most
    the quintic's largest slope (3.9 on [0, 1.2]) over the later iterations, sum_k 3.9^k < 310 over
    five; the terms' own size is at most sqrt(k) times the sum's. That is below 2^-24 x 310 x
    sqrt(k (k / 16 + 1)) / sqrt(k) = 1.9e-5 sqrt(k / 16 + 1).
  * roundings that fall to the other side because of it: no more than it again.
  * the result's own rounding: half a step (bf16 2^-8, fp32 2^-24).
"""
import ctypes
import math

import pytest

import veda_b200 as V
from tests.gpu_util import call, empty, ptr, stream, sync, torch, workspace

NS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
HALF = {V.F32: 2.0 ** -24, V.BF16: 2.0 ** -8}


def dt(dtype):
    t = torch()
    return t.float32 if dtype == V.F32 else t.bfloat16


def exact(g, steps=5, coef=NS, eps=EPS):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    a, b, c = coef
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def rounded(g, split, steps=5, coef=NS, eps=EPS):
    """The iteration with the kernels' roundings and no others."""
    t = torch()
    h = lambda v: (v * 1024).to(t.float16).double() / 1024
    two = lambda v: h(v) + h(v - h(v))
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = two(x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps))
    op = two if split else h
    a, b, c = coef
    eye = t.eye(x.shape[-2], dtype=t.float64, device=x.device)
    for k in range(steps):
        s = op(op(x) @ op(x).mT)
        m = op(a * eye + b * s + c * (s @ s))
        x = m @ op(x) + a * (x - op(x))
        if k < steps - 1:
            x = two(x)
    return x.mT if tall else x


def fro(v):
    return v.double().square().sum((-2, -1)).sqrt()


def bound(g, want, dtype, split, steps=5, coef=NS):
    """Per matrix, absolute."""
    k = max(g.shape[-2:])
    add = 2 * 1.9e-5 * math.sqrt(k / 16 + 1)
    return fro(rounded(g, split, steps, coef) - want) + (add + HALF[dtype]) * fro(want) + 1e-30


def orth(g, out=None, dtype=V.BF16, steps=5, coef=NS, eps=EPS, shape=None, ws=None):
    b, r, c = shape or g.shape
    out = empty((b, r, c), dtype) if out is None else out
    if ws is None:
        ws = workspace(V.lib().veda_orthogonalize_workspace(b, r, c, dtype))
    call("veda_orthogonalize", ptr(g), g.stride(1), g.stride(0), ptr(out), out.stride(1), out.stride(0), b, r, c,
         steps, *coef, eps, ptr(ws), ws.numel(), dtype, stream())
    return out


def make(b, r, c, dtype, seed=0, kind="noise"):
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    k = min(r, c, 4)
    v = t.randn(b, r, c, device="cuda", generator=g)
    low = t.randn(b, r, k, device="cuda", generator=g) @ t.randn(b, k, c, device="cuda", generator=g)
    v = {"noise": v, "spiked": v + 3 * low, "low rank": low}[kind]
    return (v * 0.01).to(dt(dtype))


SHAPES = [(1, 1, 1), (2, 1, 7), (1, 9, 1), (3, 16, 16), (2, 64, 64), (2, 192, 64), (1, 65, 300), (2, 300, 65),
          (1, 256, 256), (3, 257, 100), (1, 100, 520), (2, 520, 600), (1, 1001, 523),
          # the small form's borders: sides of 128 and 256, one past them, sides that are no multiple of 16
          (2, 128, 256), (2, 256, 128), (1, 129, 256), (1, 128, 257), (2, 128, 128), (3, 97, 111), (2, 33, 250),
          (2, 241, 17), (200, 24, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("b,r,c", SHAPES)
def test_orthogonalize(cuda, dtype, b, r, c):
    for kind in ("noise", "spiked"):
        g = make(b, r, c, dtype, seed=r + c, kind=kind)
        got, want = orth(g, dtype=dtype), exact(g)
        sync()
        off = fro(got.double() - want)
        assert bool((off <= bound(g, want, dtype, dtype == V.F32)).all()), (kind, (off / fro(want)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
def test_low_rank_matrices_do_not_grow_spurious_directions(cuda, dtype):
    # in fp32 (the values are exact in the type): what bf16 rounding of the input adds is not at issue
    g = make(2, 200, 300, V.F32, kind="low rank")
    if dtype == V.BF16:
        g = g.to(dt(dtype))
    got, want = orth(g, dtype=dtype), exact(g)
    sync()
    assert bool((fro(got.double() - want) <= bound(g, want, dtype, dtype == V.F32)).all())
    # the singular values that are there are near 1
    s = torch().linalg.svdvals(got[0].double())
    assert 0.6 < float(s[3]) and float(s[0]) < 1.3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("steps,coef", [(1, NS), (2, NS), (3, (1.875, -1.25, 0.375)), (8, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(cuda, dtype, steps, coef):
    g = make(2, 96, 160, dtype, seed=3)
    got, want = orth(g, dtype=dtype, steps=steps, coef=coef), exact(g, steps, coef)
    sync()
    assert bool((fro(got.double() - want) <= bound(g, want, dtype, dtype == V.F32, steps, coef)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("r,c", [(70, 45), (45, 70), (300, 264)])
def test_pitches_strides_and_bases(cuda, dtype, r, c):
    t = torch()
    g = make(3, r, c, dtype, seed=4)
    want = orth(g, dtype=dtype)
    wide = t.full((3, r + 2, c + 11), float("nan"), device="cuda", dtype=g.dtype)
    wide[:, 1:1 + r, 3:3 + c] = g
    out = t.full((3, r + 5, c + 9), 7.0, device="cuda", dtype=g.dtype)
    orth(wide[:, 1:1 + r, 3:3 + c], out=out[:, 2:2 + r, 1:1 + c], dtype=dtype, shape=(3, r, c))
    sync()
    assert bool((out[:, 2:2 + r, 1:1 + c] == want).all())
    out[:, 2:2 + r, 1:1 + c] = 7.0
    assert bool((out == 7).all())
    orth(g, out=g, dtype=dtype)   # in place
    sync()
    assert bool((g == want).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("r,c", [(40, 56), (300, 280)])
def test_a_matrix_does_not_depend_on_its_batch(cuda, dtype, r, c):
    t = torch()
    g = make(5, r, c, dtype, seed=5)
    g[1] = 0
    g[3, 2, 1] = float("nan")
    got = orth(g, dtype=dtype)
    one = [orth(g[k:k + 1], dtype=dtype) for k in range(5)]
    same = t.empty(4, r, c, device="cuda", dtype=g.dtype)
    call("veda_orthogonalize", ptr(g), c, 0, ptr(same), c, r * c, 4, r, c, 5, *NS, EPS,
         ptr(ws := workspace(V.lib().veda_orthogonalize_workspace(4, r, c, dtype))), ws.numel(), dtype, stream())
    sync()
    for k in (0, 1, 2, 4):
        assert bool((got[k] == one[k][0]).all())
    assert not bool(got[1].any()) and bool(got[3].isnan().any())
    assert all(bool((same[k] == got[0]).all()) for k in range(4))   # one matrix read four times


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_norms_of_any_size(cuda, scale):
    g = make(1, 60, 80, V.F32, seed=6) * scale
    got, want = orth(g, dtype=V.F32), exact(g)
    sync()
    # next to eps the matrix is shrunk by it: the planes' floor of 2^-35 meets an X of norm scale / eps
    floor = 3.4445 ** 5 * 2.0 ** -35 * math.sqrt(60 * 80)
    assert float(fro(got.double() - want)) <= float(bound(g, want, V.F32, True)) + floor


@pytest.mark.gpu
def test_repeats_on_other_streams_and_from_a_graph(cuda):
    t = torch()
    g = make(4, 300, 520, V.BF16, seed=7)
    want = orth(g)
    sync()
    outs = []
    for s in [t.cuda.Stream() for _ in range(2)]:
        s.wait_stream(t.cuda.current_stream())
        with t.cuda.stream(s):
            outs.append(orth(g))
    t.cuda.synchronize()
    assert all(bool((o == want).all()) for o in outs)
    ws = workspace(V.lib().veda_orthogonalize_workspace(4, 300, 520, V.BF16))
    src, out = t.zeros_like(g), empty(g.shape, V.BF16)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        orth(src, out=out, ws=ws)
    for k in range(2):
        src.copy_(g if k else g.flip(1))
        graph.replay()
    sync()
    assert bool((out == want).all())


# ---- the Muon step -------------------------------------------------------------------------------
def muon(master, momentum, grad, lowp, shape, stride, lr=1e-2, beta=0.9, nesterov=1, decay=0.1, scale=1.7, sumsq=None,
         max_norm=1.0, grad_scale=1.0, flags=0, ws=None):
    b, r, c = shape
    if ws is None:
        ws = workspace(V.lib().veda_muon_step_workspace(b, r, c, V.F32 if lowp is None else V.BF16))
    call("veda_muon_step", ptr(master), ptr(momentum), ptr(grad), ptr(lowp), b, r, c, stride, lr, beta, nesterov,
         decay, scale, 5, *NS, EPS, ptr(sumsq), max_norm, grad_scale, flags, ptr(ws), ws.numel(), stream())


def muon_want(master, momentum, grad, lr=1e-2, beta=0.9, nesterov=1, decay=0.1, scale=1.7, factor=1.0):
    g = grad.double() * factor
    m = momentum.double() * beta + g
    u = g + beta * m if nesterov else m
    o = exact(u)
    w = master.double() * (1 - lr * decay) - lr * scale * o
    return w, m, u, o, momentum.double().abs() + g.abs()


def muon_state(b, r, c, bf16, seed=0):
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    rnd = lambda s: t.randn(b, r, c, device="cuda", generator=g) * s
    master = rnd(0.02)
    return master, rnd(1e-3), rnd(1e-2), (master.to(t.bfloat16) if bf16 else None)


def check_muon(master, momentum, lowp, want, lr, scale, factor=1.0):
    t = torch()
    w, m, u, o, terms = want
    split = lowp is None
    # beta m + g: beta in fp32, the scaled and clipped gradient and the sum, each off by at most
    # 2^-24 of the terms (their sum may be far smaller)
    off = (momentum.double() - m).abs() / (2.0 ** -22 * terms + 1e-30)
    assert float(off.max()) <= 1.0
    # u itself is off by 3 x 2^-24 of its terms; amplified as the accumulation is (310)
    tol = lr * scale * (bound(u, o, V.F32, split) + 310 * 3 * 2.0 ** -24 * fro(o)) + 4 * 2.0 ** -24 * fro(w)
    assert bool((fro(master.double() - w) <= tol).all()), (fro(master.double() - w) / tol).max()
    if lowp is not None:
        assert bool((lowp == master.to(t.bfloat16)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("b,r,c", [(1, 1, 1), (2, 64, 64), (2, 192, 64), (3, 50, 77), (1, 77, 50), (2, 260, 520)])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_muon_step(cuda, bf16, b, r, c, nesterov):
    master, momentum, grad, lowp = muon_state(b, r, c, bf16, seed=r)
    want = muon_want(master, momentum, grad, nesterov=nesterov)
    keep = grad.clone()
    muon(master, momentum, grad, lowp, (b, r, c), r * c, nesterov=nesterov)
    sync()
    check_muon(master, momentum, lowp, want, 1e-2, 1.7)
    assert bool((grad == keep).all())


@pytest.mark.gpu
def test_muon_matrices_apart_in_an_arena(cuda):
    t = torch()
    b, r, c, gap = 3, 40, 72, 101   # an odd gap: every other matrix starts off a 16-byte boundary
    stride = r * c + gap
    master, momentum, grad, lowp = muon_state(b, r, c, True, seed=1)
    want = muon_want(master, momentum, grad)
    spread = []
    for v in (master, momentum, grad, lowp):
        a = t.full((b * stride,), 7.0, device="cuda", dtype=v.dtype)
        for k in range(b):
            a[k * stride:k * stride + r * c] = v[k].reshape(-1)
        spread.append(a)
    muon(*spread, (b, r, c), stride)
    sync()
    back = [t.stack([a[k * stride:k * stride + r * c].reshape(r, c) for k in range(b)]) for a in spread]
    check_muon(back[0], back[1], back[3], want, 1e-2, 1.7)
    for a in spread:
        for k in range(b):
            assert bool((a[k * stride + r * c:(k + 1) * stride] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("norm,factor", [(5.0, 0.5 / 2.5), (0.8, 1.0), (float("nan"), 1.0)])
def test_muon_clip_and_scale(cuda, norm, factor):
    # grad_scale 1/2: the norm after it is 2.5 or 0.4 against max_norm 0.5; a norm that is not finite
    # clips nothing
    t = torch()
    master, momentum, grad, lowp = muon_state(2, 48, 80, True, seed=2)
    want = muon_want(master, momentum, grad, factor=0.5 * factor)
    sumsq = t.tensor([norm * norm], dtype=t.float64, device="cuda")
    muon(master, momentum, grad, lowp, (2, 48, 80), 48 * 80, sumsq=sumsq, max_norm=0.5, grad_scale=0.5)
    sync()
    check_muon(master, momentum, lowp, want, 1e-2, 1.7)


# One matrix cut among the blocks of a cluster: 2 blocks with 1 column in the last, 9 of them (more than
# the portable 8), 16, the last one short, a smaller side of 1, of fewer rows than blocks, one past the
# borders on both sides, and more matrices than fit at once.
CUT = [(1, 128, 257), (2, 257, 128), (1, 100, 512), (1, 1, 300), (1, 7, 2049), (2, 64, 2048), (1, 128, 4096),
       (2, 4000, 37), (1, 113, 3841), (1, 128, 4097), (1, 129, 4096), (300, 48, 700), (40, 2500, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("b,r,c", CUT)
def test_matrices_cut_among_blocks(cuda, dtype, b, r, c):
    g = make(b, r, c, dtype, seed=r + c, kind="spiked")
    got, want = orth(g, dtype=dtype), exact(g)
    sync()
    off = fro(got.double() - want)
    assert bool((off <= bound(g, want, dtype, dtype == V.F32)).all()), (off / fro(want)).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("r,c", [(50, 1200), (1203, 70), (128, 2600)])
def test_matrices_cut_among_blocks_keep_their_place(cuda, dtype, r, c):
    t = torch()
    g = make(3, r, c, dtype, seed=14)
    g[1, 2, 1] = float("nan")
    want = orth(g, dtype=dtype)
    wide = t.full((3, r + 2, c + 11), float("nan"), device="cuda", dtype=g.dtype)
    wide[:, 1:1 + r, 3:3 + c] = g
    out = t.full((3, r + 5, c + 9), 7.0, device="cuda", dtype=g.dtype)
    orth(wide[:, 1:1 + r, 3:3 + c], out=out[:, 2:2 + r, 1:1 + c], dtype=dtype, shape=(3, r, c))
    one = orth(g[2:], dtype=dtype)
    sync()
    assert want[1].isnan().any() and not want[::2].isnan().any()
    part = out[:, 2:2 + r, 1:1 + c]
    assert bool((part == want)[::2].all()) and bool((one[0] == want[2]).all())
    part.fill_(7.0)
    assert bool((out == 7).all())
    out = empty((3, r, c), dtype)
    ws = workspace(V.lib().veda_orthogonalize_workspace(3, r, c, dtype))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        orth(g, out=out, dtype=dtype, ws=ws)
    for _ in range(3):
        out.zero_()
        graph.replay()
        sync()
        assert bool((out == want)[::2].all())
    orth(g, out=g, dtype=dtype)   # in place
    sync()
    assert bool((g == want)[::2].all())


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("b,r,c", [(2, 100, 2300), (3, 515, 33)])
def test_muon_on_matrices_cut_among_blocks(cuda, bf16, b, r, c):
    master, momentum, grad, lowp = muon_state(b, r, c, bf16)
    want = muon_want(master, momentum, grad)
    kept = [v.clone() for v in (master, momentum)]
    bad = grad.clone()
    bad[-1, -1, -1] = float("inf")
    muon(master, momentum, bad, lowp, (b, r, c), r * c, flags=2,
         sumsq=torch().full((1,), float("inf"), device="cuda", dtype=torch().float64))
    sync()
    assert bool((master == kept[0]).all()) and bool((momentum == kept[1]).all())
    muon(master, momentum, grad, lowp, (b, r, c), r * c)
    sync()
    check_muon(master, momentum, lowp, want, 1e-2, 1.7)


@pytest.mark.gpu
@pytest.mark.parametrize("b,r,c", [(1, 32, 4200), (2, 4203, 40)])
def test_muon_of_thin_matrices_keeps_the_weights_exact(cuda, b, r, c):
    # 30 to 50 singular values amplify what fp16 products round most: beside bf16 weights, too, such matrices
    # are multiplied as fp32 ones, within their bound
    master, momentum, grad, lowp = muon_state(b, r, c, True, seed=9)
    w, m, u, o, _ = muon_want(master, momentum, grad)
    muon(master, momentum, grad, lowp, (b, r, c), r * c)
    sync()
    tol = 1e-2 * 1.7 * (bound(u, o, V.F32, True) + 310 * 3 * 2.0 ** -24 * fro(o)) + 4 * 2.0 ** -24 * fro(w)
    assert bool((fro(master.double() - w) <= tol).all())
    assert bool((lowp == master.to(torch().bfloat16)).all())


@pytest.mark.gpu
def test_muon_skips_a_step_that_is_not_finite(cuda):
    t = torch()
    state = muon_state(2, 48, 80, True, seed=3)
    keep = [v.clone() for v in state]
    sumsq = t.tensor([float("inf")], dtype=t.float64, device="cuda")
    muon(*state, (2, 48, 80), 48 * 80, sumsq=sumsq, flags=2)
    sync()
    assert all(bool((a == b).all()) for a, b in zip(state, keep))
    sumsq[0] = 0.01
    muon(*state, (2, 48, 80), 48 * 80, sumsq=sumsq, flags=2)
    sync()
    check_muon(state[0], state[1], state[3], muon_want(*keep[:3]), 1e-2, 1.7)


@pytest.mark.gpu
def test_muon_steps_from_a_graph(cuda):
    t = torch()
    state = muon_state(2, 130, 96, True, seed=4)
    other = [v.clone() for v in state]
    for _ in range(3):
        muon(*state, (2, 130, 96), 130 * 96)
    ws = workspace(V.lib().veda_muon_step_workspace(2, 130, 96, V.BF16))
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        muon(*other, (2, 130, 96), 130 * 96, ws=ws)
    for _ in range(3):
        graph.replay()
    sync()
    assert all(bool((a == b).all()) for a, b in zip(state, other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("b,r,c", [(20, 260, 520), (2, 519, 267)])
def test_ragged_tiles_repeat_bit_for_bit(cuda, dtype, b, r, c):
    # warps with rows or columns past the end leave a tile early, and their next one may be of another product
    g = make(b, r, c, dtype, seed=r, kind="spiked")
    first, want = orth(g, dtype=dtype), exact(g)
    assert bool((fro(first.double() - want) <= bound(g, want, dtype, dtype == V.F32)).all())
    for _ in range(8):
        assert bool((orth(g, dtype=dtype) == first).all())
    state = muon_state(b, r, c, dtype == V.BF16, seed=c)
    other = [None if v is None else v.clone() for v in state]
    muon(*state, (b, r, c), r * c)
    for _ in range(4):
        again = [None if v is None else v.clone() for v in other]
        muon(*again, (b, r, c), r * c)
        assert all(a is None or bool((a == o).all()) for a, o in zip(again, state))
    sync()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("r,c", [(20, 30), (40, 600), (300, 280), (135, 50)])
def test_zero_matrices_without_eps(cuda, dtype, r, c):
    # eps = 0 leaves nothing to divide by; in one block, cut among blocks and tiled
    t = torch()
    g = make(3, r, c, dtype, seed=21)
    g[1] = 0
    got = orth(g, dtype=dtype, eps=0.0)
    want = exact(g[::2], eps=0.0)
    sync()
    assert not bool(got[1].any()) and not bool(got.isnan().any())
    off = fro(got[::2].double() - want)
    assert bool((off <= bound(g[::2], want, dtype, dtype == V.F32)).all())
    master, momentum, grad, lowp = muon_state(3, r, c, dtype == V.BF16, seed=22)
    momentum[1], grad[1] = 0, 0
    before = master.clone()
    ws = workspace(V.lib().veda_muon_step_workspace(3, r, c, dtype))
    call("veda_muon_step", ptr(master), ptr(momentum), ptr(grad), ptr(lowp), 3, r, c, r * c, 1e-2, 0.9, 1, 0.1, 1.7, 5,
         *NS, 0.0, None, 1.0, 1.0, 0, ptr(ws), ws.numel(), stream())
    sync()
    # lr, the decay and their product in fp32, and the two roundings of w - (lr decay) w
    want = before[1].double() * (1 - 1e-2 * 0.1)
    assert bool(((master[1].double() - want).abs() <= 2 * 2.0 ** -24 * before[1].double().abs()).all())
    assert not bool(momentum[1].any()) and not bool(master.isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("r,c", [(20, 30), (40, 600), (300, 280), (1001, 523)])
@pytest.mark.parametrize("power", [-128, -110, -90, 90, 125])
def test_norms_of_any_size_without_eps(cuda, dtype, r, c, power):
    # powers of two leave every mantissa as it is, so the result has the same bits: whole numbers below 8,
    # which stay exact down to the smallest subnormals of either type and up to its largest values
    t = torch()
    g = t.randint(-7, 8, (2, r, c), device="cuda", generator=t.Generator(device="cuda").manual_seed(23))
    base = orth(g.to(dt(dtype)), dtype=dtype, eps=0.0)
    got = orth(t.ldexp(g.double(), t.tensor(float(power), device="cuda", dtype=t.float64)).to(dt(dtype)), dtype=dtype, eps=0.0)
    sync()
    assert not bool(base.isnan().any()) and bool((got == base).all())


@pytest.mark.gpu
@pytest.mark.parametrize("b,r,c", [(2, 260, 520), (1, 1001, 523), (2, 100, 2300), (1, 4203, 70), (2, 80, 96)])
def test_muon_with_fp32_products_keeps_master_weights_exact(cuda, b, r, c):
    # VEDA_MUON_FP32_PRODUCTS beside bf16 weights: the bound of fp32 weights; tiled, cut among blocks and in one
    master, momentum, grad, lowp = muon_state(b, r, c, True, seed=25)
    w, m, u, o, _ = muon_want(master, momentum, grad)
    ws = workspace(V.lib().veda_muon_step_workspace(b, r, c, V.F32))
    muon(master, momentum, grad, lowp, (b, r, c), r * c, flags=4, ws=ws)
    sync()
    tol = 1e-2 * 1.7 * (bound(u, o, V.F32, True) + 310 * 3 * 2.0 ** -24 * fro(o)) + 4 * 2.0 ** -24 * fro(w)
    assert bool((fro(master.double() - w) <= tol).all()), (fro(master.double() - w) / tol).max()
    assert bool((lowp == master.to(torch().bfloat16)).all())


def test_workspace_of_muon_with_fp32_products_without_a_gpu():
    # what serves bf16 weights is too small for them
    lib = V.lib()
    buf = ctypes.create_string_buffer(1024)
    a = (ctypes.addressof(buf) + 255) // 256 * 256
    n = lib.veda_muon_step_workspace(1, 300, 400, V.BF16)
    rc = lib.veda_muon_step(a, a, a, a, 1, 300, 400, 300 * 400, 1.0, 0.9, 1, 0.0, 1.0, 5, *NS, 1e-7, None, 1.0, 1.0, 4, a, n, None)
    assert rc == V.ERR_INVALID_ARGUMENT and "workspace" in lib.veda_last_error().decode()
    assert n < lib.veda_muon_step_workspace(1, 300, 400, V.F32)


@pytest.mark.gpu
def test_long_fp32_sums_are_as_exact_as_one_chain(cuda):
    # The tensor core truncates as it adds: a chain of two k-blocks (128 terms) of one sign falls short of its sum by a
    # constant share, and the folds that join chains round to nearest and add none. One step with a = c = 0, b = 1 is
    # S X: 64 copies of a matrix side by side have its S (the copies are scaled by 1/8, exactly) and, in every
    # copy, its S X / 8, out of 64 times the chains. What the planes of X, S and M round is formed here, so the products
    # alone are compared, in the mean over 129 x 129 elements: S and M X add one chain's share each (129 terms of M X,
    # the same in both), and a fold's 2^-24 of random sign vanishes in the mean. A quarter is allowed; with chains of
    # twice the length the share of S doubles, half as much again in all, and without folds it grows 64 times.
    t = torch()
    n = 129
    u = t.rand(1, n, n, device="cuda", generator=t.Generator(device="cuda").manual_seed(24)) + 0.5
    h = lambda v: v.to(t.float16).double()
    two = lambda v: h(v) + h(v - h(v))
    short = []
    for k in (1, 64):
        g = u.repeat(1, 1, k)
        got = orth(g, dtype=V.F32, steps=1, coef=(0.0, 1.0, 0.0), eps=0.0)
        sync()
        scale = (1024.0 / g.double().square().sum().sqrt()).float()
        x = two((g * scale).double())[0]
        m = two(x @ x.mT / 1024)
        want = m @ x / 1024 / 1024
        short.append(-float(((got[0].double() - want) / want).mean()))
    assert 0 <= short[1] <= 1.25 * short[0], short


def test_workspaces_and_refusals_without_a_gpu():
    lib = V.lib()
    size = lib.veda_orthogonalize_workspace
    # two X of two fp16 planes, S and P; beside them a double for each of 256 blocks and 3 x 64 counters a
    # matrix, in six parts rounded up to 256 bytes
    n = 28 * 2048 * 1024
    rest = 28 * (256 * 8 + 3 * 64 * 4) + 6 * 256
    assert n * 8 + 28 * 2 * 1024 * 1024 * 2 <= size(28, 2048, 1024, V.BF16) <= n * 8 + 28 * 2 * 1024 * 1024 * 2 + rest
    assert size(28, 2048, 1024, V.F32) > size(28, 2048, 1024, V.BF16) == lib.veda_muon_step_workspace(28, 2048, 1024, V.BF16)
    for bad in ((0, 4, 4), (1, 0, 4), (1, 4, 0), (-1, 4, 4), (1 << 16, 4, 4), (1, 1 << 21, 4), (1, 4, 1 << 21)):
        assert size(*bad, V.F32) == 0
    assert size(1, 4, 4, 3) == 0

    buf = ctypes.create_string_buffer(1024)
    a = (ctypes.addressof(buf) + 255) // 256 * 256

    def o(g=a, ldg=4, sg=16, out=a, ldo=4, so=16, batch=2, rows=4, cols=4, steps=5, eps=1e-7, ws=a, n=1 << 40, dtype=0):
        rc = lib.veda_orthogonalize(g, ldg, sg, out, ldo, so, batch, rows, cols, steps, *NS, eps, ws, n, dtype, None)
        return rc, lib.veda_last_error().decode()

    def m(master=a, mom=a, grad=a, batch=2, rows=4, cols=4, stride=16, lr=1.0, beta=0.9, decay=0.0, steps=5, eps=0.0,
          sumsq=None, max_norm=1.0, ws=a, n=1 << 40):
        rc = lib.veda_muon_step(master, mom, grad, None, batch, rows, cols, stride, lr, beta, 1, decay, 1.0, steps,
                                *NS, eps, sumsq, max_norm, 1.0, 0, ws, n, None)
        return rc, lib.veda_last_error().decode()

    for fn, cases in ((o, [({"dtype": 2}, "dtype"), ({"rows": -1}, "shape"), ({"cols": 1 << 30}, "shape"),
                           ({"batch": 1 << 20}, "shape"), ({"ldg": 3}, "leading"), ({"ldo": 3}, "leading"),
                           ({"so": 15}, "overlap"), ({"sg": -1}, "overlap"), ({"steps": 0}, "step"), ({"steps": 65}, "step"),
                           ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"g": None}, "null"),
                           ({"out": None}, "null"), ({"n": 100}, "workspace"), ({"ws": None}, "workspace"),
                           ({"ws": a + 16}, "workspace")]),
                      (m, [({"rows": -1}, "shape"), ({"stride": 15}, "overlap"), ({"lr": -1.0}, "learning"),
                           ({"decay": -1.0}, "learning"), ({"lr": float("nan")}, "learning"), ({"beta": 1.0}, "beta"),
                           ({"steps": 0}, "step"), ({"sumsq": a, "max_norm": 0.0}, "max_norm"),
                           ({"master": None}, "null"), ({"mom": None}, "null"), ({"grad": None}, "null"),
                           ({"n": 100}, "workspace"), ({"ws": a + 8}, "workspace")])):
        for kw, word in cases:
            rc, text = fn(**kw)
            assert rc == V.ERR_INVALID_ARGUMENT and word in text, (fn.__name__, kw, rc, text)
    for empty_shape in ({"batch": 0}, {"rows": 0}, {"cols": 0}):
        assert o(**empty_shape)[0] == V.OK and m(**empty_shape)[0] == V.OK
