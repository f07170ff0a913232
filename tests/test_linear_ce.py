"""The loss head without stored logits (veda_linear_cross_entropy_{fwd,bwd}) against its formula in
64 bits.

Tolerances are bounds on what the kernels round, per element:
  z    a tensor product of `dim` terms, 16 to an instruction: each of its dim / 16 (three times that
       for split fp32 operands) additions into the fp32 accumulator is off by at most 2^-23 of what
       has been added so far (truncation), hence (segments dim / 16 + 4) 2^-23 sum |x w|; split fp32
       operands drop lo lo and the halves below 22 bits: 3 x 2^-22 sum |x w| more.
  lse  z's, plus 2^-21 for the exponentials (2^-22 each) and their sum, plus 4 steps of 2^-24 of its
       size for the scaling by log2 e and back.
  q    the error of exp(z - lse): z's and lse's together, relative; stored in bf16 (half a step,
       2^-8, which |q| <= 1 or the exact -1 bound relative to q), or as two fp16 values of 2^13 q
       (2^-21 relative, but never finer than half of fp16's smallest step, 2^-24 / 2 / 2^13 = 2^-38).
  dx   coef sum |q| |w| times q's relative error and its own additions, plus one rounding.
  dW   the same with |x| over the rows.
"""
import ctypes

import numpy as np
import pytest

import veda_b200 as V
from tests.gpu_util import call, empty, ptr, stream, sync, torch, workspace

IGN = -100
HALF = {V.F32: 2.0 ** -24, V.BF16: 2.0 ** -8}   # half a step


def dt(t, dtype):
    return t.float32 if dtype == V.F32 else t.bfloat16


def make(rows, vocab, dim, dtype, seed=0, ignored=0.0, scale=1.0):
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    x = (t.randn(rows, dim, device="cuda", generator=g) * scale).to(dt(t, dtype))
    w = (t.randn(vocab, dim, device="cuda", generator=g) / dim ** 0.5).to(dt(t, dtype))
    tg = t.randint(0, vocab, (rows,), device="cuda", generator=g)
    if ignored:
        tg[t.rand(rows, device="cuda", generator=g) < ignored] = IGN
    return x, w, tg


def need(x, w, dtype, backward):
    al = lambda m: m.stride(0) if m.data_ptr() % 16 == 0 else 1
    return V.lib().veda_linear_cross_entropy_workspace(x.shape[0], w.shape[0], x.shape[1], al(x), al(w), dtype,
                                                       backward)


def fwd(x, w, tg, dtype, ws=None, status=None):
    rows = x.shape[0]
    row, lse, loss = (empty((k,)) for k in (rows, rows, 1))
    ws = workspace(need(x, w, dtype, 0)) if ws is None else ws
    call("veda_linear_cross_entropy_fwd", ptr(x), x.stride(0), ptr(w), w.stride(0), ptr(tg), IGN, ptr(row),
         ptr(lse), ptr(loss), rows, w.shape[0], x.shape[1], ptr(ws), ws.numel(), ptr(status), dtype, stream())
    return row, lse, loss


def bwd(x, w, tg, lse, dtype, upstream=None, dx=None, dw=None, dtype_dw=None, beta=0.0, ws=None, status=None):
    dtype_dw = dtype if dtype_dw is None else dtype_dw
    ws = workspace(need(x, w, dtype, 1)) if ws is None else ws
    call("veda_linear_cross_entropy_bwd", ptr(x), x.stride(0), ptr(w), w.stride(0), ptr(tg), IGN, ptr(lse),
         ptr(upstream), ptr(dx), dx.stride(0) if dx is not None else 0, ptr(dw),
         dw.stride(0) if dw is not None else 0, dtype_dw, beta, x.shape[0], w.shape[0], x.shape[1], ptr(ws),
         ws.numel(), ptr(status), dtype, stream())


def reference(x, w, tg, dtype, upstream=1.0):
    """The formula in 64 bits and the bounds of the module's comment."""
    t = torch()
    vocab, dim = w.shape
    used = (tg != IGN) & (tg >= 0) & (tg < vocab)
    xd = t.where(used[:, None], x.double(), 0.0)
    wd = w.double()
    at = t.where(used, tg, 0)[:, None]
    count = int(used.sum())
    z = xd @ wd.t()
    lse = t.logsumexp(z, 1)
    row = t.where(used, lse - z.gather(1, at)[:, 0], 0.0)
    coef = upstream / count if count else 0.0
    q = (z - lse[:, None]).exp()
    q.scatter_add_(1, at, t.full_like(q[:, :1], -1.0))
    q = q * used[:, None]
    split = dtype == V.F32
    seg = 3 if split else 1
    acc = lambda k: (seg * k / 16 + 4) * 2.0 ** -23 + (3 * 2.0 ** -22 if split else 0.0)
    dz = acc(dim) * (xd.abs() @ wd.abs().t()).amax(1)
    dlse = dz + 2.0 ** -21 + 4 * 2.0 ** -24 * lse.abs()
    rq = (2 * dz + dlse + 2.0 ** -22)[:, None]                  # relative, of exp(z - lse)
    p = (z - lse[:, None]).exp() * used[:, None]
    eq = p * rq + q.abs() * (2.0 ** -21 if split else HALF[V.BF16]) + used[:, None] * (2.0 ** -38 if split else 0.0)
    qa = q.abs()
    # what is added over the vocabulary in fp32 (a piece's product and the pieces' sum), then rounded
    edx = abs(coef) * (eq @ wd.abs() + (acc(vocab) + 2.0 ** -16 * 2.0 ** -8) * (qa @ wd.abs()))
    edw = abs(coef) * (eq.t() @ xd.abs() + acc(x.shape[0]) * (qa.t() @ xd.abs()))
    dx, dw = coef * (q @ wd), coef * (q.t() @ xd)
    tiny = 1e-37
    return {"used": used, "row": row, "lse": lse, "loss": row.sum() / max(count, 1), "dlse": dlse,
            "drow": t.where(used, dz + dlse + 2.0 ** -23 * row.abs(), 0.0), "dx": dx, "dw": dw,
            "edx": edx + HALF[dtype] * dx.abs() * (1 + 2.0 ** -8) + tiny,
            "edw": lambda out: edw + HALF[out] * dw.abs() * (1 + 2.0 ** -8) + tiny}


def within(got, want, tol, what):
    off = (got.double() - want).abs()
    assert not bool(got.isnan().any()), f"{what}: NaN"
    bad = off > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.2f} bounds"


def run_and_check(x, w, tg, dtype, dtype_dw=None):
    dtype_dw = dtype if dtype_dw is None else dtype_dw
    r = reference(x, w, tg, dtype)
    row, lse, loss = fwd(x, w, tg, dtype)
    dx, dw = empty(x.shape, dtype), empty(w.shape, dtype_dw)
    bwd(x, w, tg, lse, dtype, dx=dx, dw=dw, dtype_dw=dtype_dw)
    sync()
    u = r["used"]
    within(lse[u], r["lse"][u], r["dlse"][u], "lse")
    within(row, r["row"], r["drow"] + 1e-30, "row loss")
    assert abs(float(loss) - float(r["loss"])) <= float(r["drow"].max()) + 2.0 ** -23 * abs(float(r["loss"]))
    within(dx, r["dx"], r["edx"], "dx")
    within(dw, r["dw"], r["edw"](dtype_dw), "dw")
    return row, lse, loss, dx, dw


SHAPES = [(1, 1, 8), (1, 300, 64), (3, 2, 16), (31, 255, 24), (128, 512, 64), (257, 256, 40), (200, 1000, 256),
          (300, 257, 72), (512, 2049, 128), (77, 5001, 520), (1030, 770, 136),
          # up to four rows of up to 2048 columns are streamed past; one past each border
          (2, 700, 2048), (3, 601, 1000), (4, 9001, 776), (5, 4100, 64), (4, 50, 2056), (1, 20000, 40), (4, 33, 1),
          (8, 9001, 776),
          # the tensor-core form: over 1024 rows, 4096 words (bf16: 1024) or 2^23 products (bf16: 2^22)
          (31, 4355, 24), (128, 5000, 64), (257, 4353, 40), (300, 4097, 72), (512, 6145, 128), (1025, 255, 16),
          (9, 4111, 8), (700, 4000, 100), (1024, 4096, 8),
          # small gradients cut into 1, 2, 4 and 8 parts, the last parts short or empty
          (5, 129, 40), (130, 257, 33), (300, 40, 64), (513, 150, 90), (1024, 33, 100), (9, 1153, 500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab,dim", SHAPES)
def test_loss_and_gradients(cuda, dtype, rows, vocab, dim):
    run_and_check(*make(rows, vocab, dim, dtype, seed=rows + vocab, ignored=0.2 if rows > 2 else 0.0), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,vocab,dim", [(V.BF16, 5000, 15000, 64), (V.F32, 2500, 10000, 64)])
def test_many_pieces_of_the_vocabulary(cuda, dtype, rows, vocab, dim):
    # the pieces of q are 64 MB: 6656 columns at 5000 bf16 rows or 2500 split ones
    run_and_check(*make(rows, vocab, dim, dtype, seed=5, ignored=0.1), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 3001, 116), (2, 1037, 102), (3, 515, 101), (4, 40, 260), (1, 9, 2046),
                                             (4, 2000, 1999), (1, 200, 4), (20, 511, 118), (9, 300, 61)])
def test_rows_of_every_alignment(cuda, dtype, rows, vocab, dim):
    # head and dW in groups of 8, 4, 2 and single elements: by dim, by pitch, by base
    t = torch()
    x, w, tg = make(rows, vocab, dim, dtype, seed=dim)
    for pitch, base in ((dim, 0), (dim + dim % 2, 0), ((dim + 7) // 8 * 8, 0), ((dim + 7) // 8 * 8, 4), (dim + 6, 2), (dim + 1, 1)):
        ww = t.full((vocab * pitch + base + 8,), float("nan"), device="cuda", dtype=w.dtype)
        wv = ww[base:base + vocab * pitch].view(vocab, pitch)[:, :dim]
        wv.copy_(w)
        run_and_check(x, wv, tg, dtype)
    # dW in rows of 16-byte pitch whose last columns are no whole group, its padding untouched
    pitch = (dim + 7) // 8 * 8 + 8
    _, lse, _ = fwd(x, w, tg, dtype)
    want, wide = empty(w.shape, dtype), t.full((vocab, pitch), 7.0, device="cuda", dtype=w.dtype)
    bwd(x, w, tg, lse, dtype, dx=None, dw=want, dtype_dw=dtype)
    bwd(x, w, tg, lse, dtype, dx=None, dw=wide[:, :dim], dtype_dw=dtype)
    sync()
    assert bool((wide[:, :dim] == want).all()) and bool((wide[:, dim:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab,dim", [(65, 130, 7), (40, 300, 100), (129, 257, 33), (4, 300, 100), (2, 1001, 33), (65, 4130, 7),
                                             (300, 4300, 100), (1029, 257, 33)])
def test_odd_widths_pitches_and_bases(cuda, dtype, rows, vocab, dim):
    t = torch()
    x, w, tg = make(rows, vocab, dim, dtype, seed=2)
    run_and_check(x, w, tg, dtype)
    wide = t.full((rows, dim + 13), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, 5:5 + dim] = x
    ww = t.full((vocab, dim + 3), float("nan"), device="cuda", dtype=x.dtype)
    ww[:, 1:1 + dim] = w
    xs, wv = wide[:, 5:5 + dim], ww[:, 1:1 + dim]
    a = run_and_check(xs, wv, tg, dtype)
    b = run_and_check(x, w, tg, dtype)
    assert all(bool((p == q).all()) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("vocab", [500, 4500])
def test_aligned_slices_are_read_in_place_and_padding_stays(cuda, dtype, vocab):
    t = torch()
    rows, dim = 100, 64
    x, w, tg = make(rows, vocab, dim, dtype, seed=3)
    wide = t.full((rows, 192), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, 64:128] = x
    r = reference(x, w, tg, dtype)
    _, lse, _ = fwd(wide[:, 64:128], w, tg, dtype)
    gx = t.full((rows + 3, 80), 7.0, device="cuda", dtype=x.dtype)
    gw = t.full((vocab + 3, 96), 7.0, device="cuda", dtype=w.dtype)
    bwd(wide[:, 64:128], w, tg, lse, dtype, dx=gx[:rows, 8:72], dw=gw[:vocab, 16:80])
    sync()
    within(gx[:rows, 8:72], r["dx"], r["edx"], "dx")
    within(gw[:vocab, 16:80], r["dw"], r["edw"](dtype), "dw")
    assert bool((gx[rows:] == 7).all() and (gx[:, :8] == 7).all() and (gx[:, 72:] == 7).all())
    assert bool((gw[vocab:] == 7).all() and (gw[:, :16] == 7).all() and (gw[:, 80:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dtype_dw", [(V.BF16, V.BF16), (V.BF16, V.F32), (V.F32, V.F32)])
@pytest.mark.parametrize("pitch", [64, 67])
@pytest.mark.parametrize("rows,vocab", [(150, 700), (3, 700), (150, 4700)])
def test_accumulated_weight_gradient_and_upstream(cuda, dtype, dtype_dw, pitch, rows, vocab):
    t = torch()
    dim = 64
    x, w, tg = make(rows, vocab, dim, dtype, seed=4, ignored=0.3)
    up = t.tensor([-2.5], device="cuda")
    r = reference(x, w, tg, dtype, upstream=-2.5)
    _, lse, _ = fwd(x, w, tg, dtype)
    base = t.randn(vocab, pitch, device="cuda").to(dt(t, dtype_dw))
    got = base.clone()
    dx = empty(x.shape, dtype)
    bwd(x, w, tg, lse, dtype, upstream=up, dx=dx, dw=got[:, :dim], dtype_dw=dtype_dw, beta=1.0)
    sync()
    want = base[:, :dim].double() + r["dw"]
    within(dx, r["dx"], r["edx"], "dx")
    within(got[:, :dim], want, r["edw"](V.F32) + HALF[dtype_dw] * want.abs() * 1.01, "dw")
    assert bool((got[:, dim:] == base[:, dim:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab", [(200, 1500), (4, 1500), (300, 5500)])
def test_one_gradient_alone_has_the_bits_of_both(cuda, dtype, rows, vocab):
    x, w, tg = make(rows, vocab, 96, dtype, seed=6)
    _, lse, _ = fwd(x, w, tg, dtype)
    dx, dw, dx1, dw1 = empty(x.shape, dtype), empty(w.shape, dtype), empty(x.shape, dtype), empty(w.shape, dtype)
    bwd(x, w, tg, lse, dtype, dx=dx, dw=dw)
    bwd(x, w, tg, lse, dtype, dx=dx1)
    bwd(x, w, tg, lse, dtype, dw=dw1)
    bwd(x, w, tg, lse, dtype)
    sync()
    assert bool((dx == dx1).all()) and bool((dw == dw1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab", [(200, 600), (4, 600), (200, 4600)])
def test_padding_that_holds_nan_reaches_nothing(cuda, dtype, rows, vocab):
    t = torch()
    x, w, tg = make(rows, vocab, 64, dtype, seed=7)
    tg[::2] = IGN
    clean = x.clone()
    for k, v in enumerate((float("nan"), float("inf"), -float("inf"), 3e38)):
        x[2 * k % rows] = v
    _, lse, loss = fwd(x, w, tg, dtype)
    row, lse0, loss0 = fwd(clean, w, tg, dtype)
    got = [empty(x.shape, dtype), empty(w.shape, dtype)]
    want = [empty(x.shape, dtype), empty(w.shape, dtype)]
    bwd(x, w, tg, lse, dtype, dx=got[0], dw=got[1])
    bwd(clean, w, tg, lse0, dtype, dx=want[0], dw=want[1])
    sync()
    used = tg != IGN
    assert float(loss) == float(loss0) and bool((lse[used] == lse0[used]).all()) and bool((row[~used] == 0).all())
    assert all(bool((a == b).all()) for a, b in zip(got, want)) and bool((got[0][~used] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("rows,vocab", [(50, 300), (3, 300), (50, 4300)])
def test_no_counted_row(cuda, dtype, rows, vocab):
    x, w, tg = make(rows, vocab, 32, dtype, seed=8)
    tg[:] = IGN
    row, lse, loss = fwd(x, w, tg, dtype)
    dx, dw = empty(x.shape, dtype), empty(w.shape, dtype)
    bwd(x, w, tg, lse, dtype, dx=dx, dw=dw)
    sync()
    assert float(loss) == 0.0 and not bool(row.any()) and not bool(dx.any()) and not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 300, 1 << 40])
@pytest.mark.parametrize("rows,vocab", [(60, 300), (4, 300), (60, 4300)])
def test_target_outside_the_vocabulary_sets_the_status_and_is_not_counted(cuda, bad, rows, vocab):
    t = torch()
    x, w, tg = make(rows, vocab, 32, V.BF16, seed=9)
    bad = vocab if bad == 300 else bad
    want = tg.clone()
    want[3] = IGN
    tg[3] = bad
    status = t.zeros(1, dtype=t.int32, device="cuda")
    row, lse, loss = fwd(x, w, tg, V.BF16, status=status)
    sync()
    assert int(status) == V.ERR_OUT_OF_RANGE
    status.zero_()
    dx, dw, dx0, dw0 = (empty(s.shape, V.BF16) for s in (x, w, x, w))
    bwd(x, w, tg, lse, V.BF16, dx=dx, dw=dw, status=status)
    assert int(status) == V.ERR_OUT_OF_RANGE
    status.zero_()
    _, lse0, loss0 = fwd(x, w, want, V.BF16, status=status)
    bwd(x, w, want, lse0, V.BF16, dx=dx0, dw=dw0, status=status)
    sync()
    assert int(status) == 0 and float(loss) == float(loss0) and bool((dx == dx0).all()) and bool((dw == dw0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
def test_large_logits(cuda, dtype):
    # logits of several hundred: exp of them overflows, of their differences does not
    run_and_check(*make(90, 700, 64, dtype, seed=10, scale=150.0), dtype)
    run_and_check(*make(90, 4700, 64, dtype, seed=10, scale=150.0), dtype)


@pytest.mark.gpu
def test_fp32_operands_of_any_magnitude(cuda):
    # 2^100 on one side and 2^-100 on the other leave the logits as they are; the gradients scale
    t = torch()
    x, w, tg = make(60, 4300, 48, V.F32, seed=11)
    base = run_and_check(x, w, tg, V.F32)
    big = (x * 2.0 ** 100, w * 2.0 ** -100)
    row, lse, loss = fwd(*big, tg, V.F32)
    dx, dw = empty(x.shape), empty(w.shape)
    bwd(*big, tg, lse, V.F32, dx=dx, dw=dw)
    sync()
    assert bool((lse == base[1]).all()) and bool((row == base[0]).all())
    assert bool((dx * 2.0 ** 100 == base[3]).all()) and bool((dw * 2.0 ** -100 == base[4]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(40, 200), (4, 200), (40, 4200)])
def test_gradients_against_differences(cuda, rows, vocab):
    t = torch()
    x, w, tg = make(rows, vocab, 32, V.F32, seed=12, ignored=0.2)
    _, lse, _ = fwd(x, w, tg, V.F32)
    dx, dw = empty(x.shape), empty(w.shape)
    bwd(x, w, tg, lse, V.F32, dx=dx, dw=dw)
    g = t.Generator(device="cuda").manual_seed(1)
    h = 2.0 ** -5
    loss64 = lambda a, b: float(reference(a, b, tg, V.F32)["loss"])
    for k in range(4):
        ux = t.randn(x.shape, device="cuda", generator=g)
        uw = t.randn(w.shape, device="cuda", generator=g) * 0.2
        up, down = (x + h * ux, w + h * uw), (x - h * ux, w - h * uw)
        diff = (float(fwd(*up, tg, V.F32)[2]) - float(fwd(*down, tg, V.F32)[2])) / (2 * h)
        slope = float((dx.double() * ux).sum() + (dw.double() * uw).sum())
        # the difference quotient's own error, measured in 64 bits, and the losses' rounding over 2 h
        r = reference(x, w, tg, V.F32)
        true = float((r["dx"] * ux).sum() + (r["dw"] * uw).sum())
        trunc = abs((loss64(*up) - loss64(*down)) / (2 * h) - true)
        tol = trunc + 2 * float(r["drow"].max()) / h + float((r["edx"] * ux.abs()).sum() + (r["edw"](V.F32) * uw.abs()).sum())
        assert abs(diff - slope) <= tol, (diff, slope, tol)
    sync()


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_other_streams_and_from_a_graph(cuda):
    t = torch()
    x, w, tg = make(700, 9000, 128, V.BF16, seed=13, ignored=0.1)
    _, lse, loss = fwd(x, w, tg, V.BF16)
    dx, dw = empty(x.shape, V.BF16), empty(w.shape, V.BF16)
    bwd(x, w, tg, lse, V.BF16, dx=dx, dw=dw)
    sync()
    side = [t.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:   # two calls at once, each with its own workspace
        s.wait_stream(t.cuda.current_stream())
        with t.cuda.stream(s):
            _, l2, loss2 = fwd(x, w, tg, V.BF16)
            a, b = empty(x.shape, V.BF16), empty(w.shape, V.BF16)
            bwd(x, w, tg, l2, V.BF16, dx=a, dw=b)
            outs.append((l2, loss2, a, b))
    t.cuda.synchronize()
    for l2, loss2, a, b in outs:
        assert bool((l2 == lse).all()) and float(loss2) == float(loss) and bool((a == dx).all()) and bool((b == dw).all())
    ws = workspace(max(need(x, w, V.BF16, k) for k in (0, 1)))
    row, l3, loss3 = empty((700,)), empty((700,)), empty((1,))
    a, b = empty(x.shape, V.BF16), empty(w.shape, V.BF16)
    graph = t.cuda.CUDAGraph()
    xin = x.clone()
    with t.cuda.graph(graph):
        call("veda_linear_cross_entropy_fwd", ptr(xin), 128, ptr(w), 128, ptr(tg), IGN, ptr(row), ptr(l3), ptr(loss3),
             700, 9000, 128, ptr(ws), ws.numel(), None, V.BF16, stream())
        bwd(xin, w, tg, l3, V.BF16, dx=a, dw=b, ws=ws)
    for k in range(2):
        xin.copy_(x if k else x * 2)
        graph.replay()
    sync()
    assert bool((l3 == lse).all()) and bool((a == dx).all()) and bool((b == dw).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("scale", [2.0 ** 7, 1e6, 1e-30])
@pytest.mark.parametrize("rows,vocab,dim", [(4, 300, 64), (60, 300, 64), (60, 4300, 64), (300, 5001, 40)])
@pytest.mark.parametrize("counted", [0.5, 0.0])
def test_lse_of_rows_that_are_not_counted(cuda, dtype, scale, rows, vocab, dim, counted):
    # lse is every row's, whatever the others hold: rows that are not counted far above or below the counted
    # ones in size, and no counted row at all
    t = torch()
    x, w, tg = make(rows, vocab, dim, dtype, seed=15)
    clean = x.clone()
    if counted:
        tg[1::2] = IGN
    else:
        tg[:] = IGN
    x[1::2] = (x[1::2].float() * scale).to(x.dtype)
    row, lse, loss = fwd(x, w, tg, dtype)
    row0, lse0, loss0 = fwd(clean, w, tg, dtype)
    sync()
    # the module's bounds, every row's own
    z = x.double() @ w.double().t()
    seg, drop = (3, 3 * 2.0 ** -22) if dtype == V.F32 else (1, 0.0)
    dz = ((seg * dim / 16 + 4) * 2.0 ** -23 + drop) * (x.double().abs() @ w.double().abs().t()).amax(1)
    want = t.logsumexp(z, 1)
    within(lse, want, dz + 2.0 ** -21 + 4 * 2.0 ** -24 * want.abs(), "lse")
    assert bool((row[tg == IGN] == 0).all())
    assert bool((row == row0).all()) and float(loss) == float(loss0) and bool((lse[::2] == lse0[::2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [V.BF16, V.F32])
@pytest.mark.parametrize("scale", [1e9, 1e14, 1e30])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 300, 64), (4, 300, 64), (60, 300, 64), (60, 4300, 64), (300, 5001, 40)])
def test_forward_of_huge_logits(cuda, dtype, scale, rows, vocab, dim):
    # logits whose rounding in log2 units is itself past the exponential's range: the reference of a row's sum lies
    # above them, so no term overflows, and a sum that vanishes leaves the maximum
    t = torch()
    x, w, tg = make(rows, vocab, dim, dtype, seed=19, ignored=0.2)
    x = (x.float() * scale).to(x.dtype)
    row, lse, loss = fwd(x, w, tg, dtype)
    sync()
    z = x.double() @ w.double().t()
    seg, drop = (3, 3 * 2.0 ** -22) if dtype == V.F32 else (1, 0.0)
    dz = ((seg * dim / 16 + 4) * 2.0 ** -23 + drop) * (x.double().abs() @ w.double().abs().t()).amax(1)
    want = t.logsumexp(z, 1)
    # beside the module's bounds: a sum of up to `vocab` terms that vanished against the maximum's rounding
    dlse = dz + 2.0 ** -21 + 4 * 2.0 ** -24 * want.abs() + t.where(want.abs() > 1e9, float(np.log(vocab)), 0.0)
    within(lse, want, dlse, "lse")
    used = tg != IGN
    at = t.where(used, tg, 0)[:, None]
    drow = dz + dlse + 2.0 ** -23 * (want.abs() + z.gather(1, at)[:, 0].abs())
    within(row, t.where(used, want - z.gather(1, at)[:, 0], 0.0), t.where(used, drow, 0.0) + 1e-30, "row loss")
    assert bool(loss.isfinite().all())


def _bias(got, want):
    return float(((got.double() - want) / want).mean())


@pytest.mark.gpu
def test_long_fp32_sums_are_as_exact_as_one_chain(cuda):
    # The tensor core truncates as it adds, so what a chain of four k-blocks (256 terms) falls short of its sum
    # is a constant share of it where all terms have one sign; the folds that join the chains round to nearest
    # and add none. 32 times the same terms therefore fall short by the same share as 256 do: in the mean over
    # 1024 columns the folds' own roundings (half of 2^-24 rms, 32 of them, of sums that grow evenly) leave 3e-9, and
    # 1e-7 is allowed. A chain of twice the length would add 8 more additions of half of 2^-24 or so each, 2e-7 and
    # more, one without folds a hundred times that. Logits of 0 and one lse for all rows make every q the same
    # number, exp(-0.3) (with all its bits in use), and its own rounding the same in both; the target's word or row
    # holds zeros.
    t = torch()
    dim, rows, words = 1024, 8192, 256
    g = t.Generator(device="cuda").manual_seed(16)
    lse = t.full((rows,), 0.3, device="cuda")
    q = float(np.exp(-float(np.float32(0.3))))
    tg = t.zeros(rows, device="cuda", dtype=t.int64)
    short = []
    for k in (1, 32):
        w = t.rand(words, dim, device="cuda", generator=g.manual_seed(17)) + 0.5
        w[0] = 0
        w = w.repeat(k, 1)
        dx = empty((rows, dim))
        bwd(t.zeros(rows, dim, device="cuda"), w, tg, lse, V.F32, dx=dx)
        sync()
        assert bool((dx == dx[0]).all())
        short.append(-_bias(dx[0], q * w.double().sum(0) / rows))
    assert abs(short[1] - short[0]) <= 1e-7, short
    short = []
    for k in (1, 32):
        n = words * k
        x = (t.rand(words, dim, device="cuda", generator=g.manual_seed(18)) + 0.5).repeat(k, 1)
        dw = empty((4500, dim))
        bwd(x, t.zeros(4500, dim, device="cuda"), tg[:n], lse[:n], V.F32, dw=dw)
        sync()
        assert bool((dw[1:] == dw[1]).all())
        short.append(-_bias(dw[1], q * x.double().sum(0) / n))
    assert abs(short[1] - short[0]) <= 1e-7, short


def test_workspace_sizes_and_refusals_without_a_gpu():
    lib = V.lib()
    size = lib.veda_linear_cross_entropy_workspace
    # pieces of q stay near 128 MB in all whatever the rows, unless one 256-column piece is larger
    for rows in (1, 100, 8192, 30000):
        assert 0 < size(rows, 151936, 1024, 1024, 1024, V.BF16, 1) <= (130 << 20) + rows * 1024 * 6 + (1 << 20)
    assert size(8192, 151936, 1024, 1024, 1024, V.BF16, 0) < 32 << 20
    # an operand that cannot be read in place is laid out in the workspace (not in the small form: few words)
    assert size(64, 5000, 100, 100, 104, V.BF16, 0) - size(64, 5000, 100, 104, 104, V.BF16, 0) >= 64 * 104 * 2
    assert size(64, 5000, 100, 104, 100, V.BF16, 0) - size(64, 5000, 100, 104, 104, V.BF16, 0) >= 5000 * 104 * 2
    for bad in ((0, 5, 8), (5, 0, 8), (5, 5, 0), (-1, 5, 8), (1 << 40, 5, 8)):
        assert size(*bad, 8, 8, V.BF16, 1) == 0
    assert size(5, 5, 8, 8, 8, 7, 0) == 0

    buf = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(buf) + 255) // 256 * 256

    def f(x=a, ldx=8, w=a, ldw=8, t=a, row=a, rows=4, vocab=5, dim=8, ws=a, n=0, dtype=V.BF16):
        rc = lib.veda_linear_cross_entropy_fwd(x, ldx, w, ldw, t, IGN, row, None, None, rows, vocab, dim, ws, n,
                                               None, dtype, None)
        return rc, lib.veda_last_error().decode()

    def b(x=a, ldx=8, w=a, ldw=8, t=a, lse=a, dx=a, lddx=8, dw=a, lddw=8, ddw=V.BF16, beta=0.0, rows=4, vocab=5,
          dim=8, ws=a, n=0, dtype=V.BF16):
        rc = lib.veda_linear_cross_entropy_bwd(x, ldx, w, ldw, t, IGN, lse, None, dx, lddx, dw, lddw, ddw, beta,
                                               rows, vocab, dim, ws, n, None, dtype, None)
        return rc, lib.veda_last_error().decode()

    for fn in (f, b):
        for kw, word in (({"dtype": 5}, "dtype"), ({"rows": -1}, "shape"), ({"vocab": 0}, "shape"),
                         ({"dim": 0}, "shape"), ({"ldx": 7}, "leading"), ({"ldw": 7}, "leading"),
                         ({"x": None}, "null"), ({"w": None}, "null"), ({"t": None}, "null"),
                         ({"n": 10}, "workspace"), ({"ws": None, "n": 1 << 40}, "workspace"),
                         ({"ws": a + 8, "n": 1 << 40}, "workspace"), ({"rows": 1 << 40}, "31 bits")):
            rc, text = fn(**kw)
            assert rc == V.ERR_INVALID_ARGUMENT and word in text, (fn.__name__, kw, rc, text)
    assert f(row=None)[0] == V.ERR_INVALID_ARGUMENT
    for kw, word in (({"lse": None}, "null"), ({"lddx": 7}, "leading"), ({"lddw": 7}, "leading"),
                     ({"beta": 0.5}, "beta_dw"), ({"ddw": 9}, "dtype"),
                     ({"dtype": V.F32, "ddw": V.BF16}, "fp32 weight gradient")):
        rc, text = b(**kw)
        assert rc == V.ERR_INVALID_ARGUMENT and word in text, (kw, rc, text)
    # nothing asked for: nothing done
    assert b(dx=None, dw=None)[0] == V.OK and b(rows=0, dx=None, dw=None)[0] == V.OK
    assert f(rows=0)[0] == V.OK
