"""The two ends of the backward pass as operators, measured: the loss head and the optimiser.

  linear cross-entropy   the LM head's product and its softmax cross-entropy in one operator that
                         never stores the [rows, vocab] logits, forward and with its gradients
  orthogonalise          a batch of matrices to (nearly) orthogonal ones by Newton-Schulz products
  Muon step              momentum, orthogonalised update and decoupled weight decay of a batch of
                         weight matrices

With own = False, run() computes each from elementary torch operations in 32 bits; with own = True
it calls the library's entry points (include/veda_cuda.h). A state is what a training program holds:
the hidden rows, the head, the targets; or the gradients, momentum, master weights and weights.
"""
from __future__ import annotations

import math

import torch

own = False

IGNORE = -100                       # the target of a padded row
NS = (3.4445, -4.7750, 2.0315)      # the quintic's coefficients, as Muon uses them
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, DECAY = 3e-4, 0.95, 0.1


def _loss(name, dtype, rows, vocab, dim, grads, ignored=0.0, pitch=0):
    return {"name": name, "op": "loss", "dtype": dtype, "rows": rows, "vocab": vocab, "dim": dim,
            "grads": grads, "ignored": ignored, "pitch": pitch}


def _mat(name, op, dtype, batch, rows, cols):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "rows": rows, "cols": cols}


def listed():
    return [
        # the tiny fp32 decoder's step: 4 x 32 tokens, all launch latency
        _loss("loss_step_tiny_f32", "f32", 128, 512, 64, True),
        # an fp32 head of odd sizes with a padded batch
        _loss("loss_step_odd_f32", "f32", 1000, 10007, 320, True, 0.2),
        # the score of one token under the 0.6B head: the head is read once
        _loss("loss_one_row", "bf16", 1, 151936, 1024, False),
        # the evaluation of one 2048-token sequence: the loss alone
        _loss("loss_eval", "bf16", 2048, 151936, 1024, False),
        # a padded batch with a prime vocabulary, hidden rows that are a slice of a wider buffer
        _loss("loss_step_padded", "bf16", 1237, 50021, 768, True, 0.3, 1024),
        # the 0.6B training step's head: 4 x 2048 tokens
        _loss("loss_step", "bf16", 8192, 151936, 1024, True),
        # the tiny decoder's up projections
        _mat("orth_tiny_f32", "orth", "f32", 2, 192, 64),
        # one odd fp32 matrix
        _mat("orth_odd_f32", "orth", "f32", 1, 1001, 523),
        # the k projections of every layer of the 0.6B decoder
        _mat("orth_square", "orth", "bf16", 28, 1024, 1024),
        # the tiny decoder's output projections, fp32 weights
        _mat("muon_tiny_f32", "muon", "f32", 2, 64, 64),
        # the q projections of every layer of the 0.6B decoder
        _mat("muon_tall", "muon", "bf16", 28, 2048, 1024),
        # down projections of the 1.7B decoder, eight layers
        _mat("muon_wide", "muon", "bf16", 8, 2048, 6144),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("loss", "loss", "orth", "muon"))
    if op == "loss":
        dtype = rng.choice(("bf16", "bf16", "f32"))
        top = 8192 * 151936 * 1024 if dtype == "bf16" else 1000 * 10007 * 320
        while True:
            rows = _log(rng, 1, 8192)
            vocab = _log(rng, 512, 151936 if dtype == "bf16" else 20000)
            dim = _log(rng, 64, 2048 if dtype == "bf16" else 512)
            if rng.random() < 0.7:
                dim = dim // 8 * 8
            if rows * vocab * dim <= top:
                break
        c = _loss("", dtype, rows, vocab, dim, rng.random() < 0.7, rng.choice((0.0, 0.1, 0.5)),
                  rng.choice((0, dim + rng.randrange(1, 64))))
    else:
        dtype = rng.choice(("bf16", "bf16", "f32"))
        while True:
            batch = _log(rng, 1, 28)
            rows, cols = _log(rng, 16, 6144), _log(rng, 16, 6144)
            top = _ns_flops(8, 2048, 6144) / (1 if dtype == "bf16" else 8)
            if _ns_flops(batch, rows, cols) <= top and batch * rows * cols <= 8 * 2048 * 6144:
                break
        c = _mat("", op, dtype, batch, rows, cols)
    del c["name"]
    return c


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _type(case)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "loss":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        w = (randn(v, d) * 0.02).to(dt)
        t = torch.randint(0, v, (n,), device="cuda", generator=g)
        # normed hidden rows; half of them lean towards their target's row, as a trained model's do
        lean = (torch.rand(n, 1, device="cuda", generator=g) < 0.5) * (5.0 / (0.0004 * d))
        x = (randn(n, d) + lean * w[t].float()).to(dt)
        if case["pitch"]:
            wide = torch.zeros(n, case["pitch"], device="cuda", dtype=dt)
            wide[:, :d] = x
            x = wide[:, :d]
        if case["ignored"]:
            t[torch.rand(n, device="cuda", generator=g) < case["ignored"]] = IGNORE
        return {"case": dict(case), "x": x, "w": w, "t": t}
    b, r, c = case["batch"], case["rows"], case["cols"]
    # gradients of few directions that dominate, over noise
    k = min(8, r, c)
    grad = randn(b, r, k) @ randn(b, k, c) * (0.05 / math.sqrt(k)) + randn(b, r, c) * 0.05
    if case["op"] == "orth":
        return {"case": dict(case), "g": grad.to(dt)}
    master = randn(b, r, c) * 0.02
    if dt == torch.bfloat16:
        lowp = master.to(dt)
    else:
        lowp = None
    return {"case": dict(case), "g": grad * 1e-3, "momentum": randn(b, r, c) * 1e-3, "master": master,
            "lowp": lowp}


# ---- plain forms -------------------------------------------------------------------------------
def _plain_loss(s):
    c = s["case"]
    x, w, t = s["x"].float(), s["w"].float(), s["t"]
    used = t != IGNORE
    at = torch.where(used, t, 0)[:, None]
    count = used.sum().clamp(min=1)
    z = x @ w.t()
    top = z.amax(1)
    lse = top + (z - top[:, None]).exp().sum(1).log()
    row = torch.where(used, lse - z.gather(1, at)[:, 0], 0.0)
    out = {"loss": row.double().sum().div(count).float(), "row_loss": row, "lse": lse}
    if c["grads"]:
        p = (z - lse[:, None]).exp()
        del z
        p.scatter_add_(1, at, torch.full_like(p[:, :1], -1.0))
        p *= (used / count)[:, None]
        out["dx"] = (p @ w).to(s["x"].dtype)
        out["dw"] = (p.t() @ x).to(s["w"].dtype)
    return out


def _plain_orth(g, steps=STEPS):
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = NS
    for _ in range(steps):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(1, 2) if tall else x


def _plain_muon(s):
    g, m, w = s["g"], s["momentum"], s["master"]
    m.mul_(MOMENTUM).add_(g)
    u = _plain_orth(g + MOMENTUM * m)
    w.copy_(w - LR * DECAY * w - LR * _update_scale(s["case"]) * u)
    if s["lowp"] is not None:
        s["lowp"].copy_(w)


def _update_scale(case):
    return 0.2 * math.sqrt(max(case["rows"], case["cols"]))


# ---- the library's entry points ----------------------------------------------------------------
def _lib():
    import veda_b200
    return veda_b200, veda_b200.lib(), torch.cuda.current_stream().cuda_stream


def _own_loss(s):
    veda, lib, stream = _lib()
    c = s["case"]
    n, v, d = c["rows"], c["vocab"], c["dim"]
    x, w, t = s["x"], s["w"], s["t"]
    dt = veda.F32 if c["dtype"] == "f32" else veda.BF16
    if "work" not in s:   # the workspace a training program keeps
        size = max(lib.veda_linear_cross_entropy_workspace(n, v, d, x.stride(0), w.stride(0), dt, k)
                   for k in range(1 + c["grads"]))
        s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    stats = torch.empty(2 * n + 1, device="cuda")
    row, lse, loss = stats[:n], stats[n:2 * n], stats[2 * n]
    work = s["work"]
    veda.check(lib.veda_linear_cross_entropy_fwd(
        x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), t.data_ptr(), IGNORE, row.data_ptr(),
        lse.data_ptr(), loss.data_ptr(), n, v, d, work.data_ptr(), work.numel(), None, dt, stream))
    out = {"loss": loss, "row_loss": row, "lse": lse}
    if c["grads"]:
        dx = torch.empty(n, d, dtype=x.dtype, device="cuda")
        dw = torch.empty(v, d, dtype=w.dtype, device="cuda")
        veda.check(lib.veda_linear_cross_entropy_bwd(
            x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), t.data_ptr(), IGNORE,
            lse.data_ptr(), None, dx.data_ptr(), d, dw.data_ptr(), d, dt, 0.0, n, v, d,
            work.data_ptr(), work.numel(), None, dt, stream))
        out["dx"], out["dw"] = dx, dw
    return out


def _own_orth(s):
    veda, lib, stream = _lib()
    c, g = s["case"], s["g"]
    b, r, k = c["batch"], c["rows"], c["cols"]
    dt = veda.F32 if c["dtype"] == "f32" else veda.BF16
    if "work" not in s:
        s["work"] = torch.empty(lib.veda_orthogonalize_workspace(b, r, k, dt), dtype=torch.uint8,
                                device="cuda")
    out = torch.empty_like(g)
    veda.check(lib.veda_orthogonalize(g.data_ptr(), k, r * k, out.data_ptr(), k, r * k, b, r, k, STEPS,
                                      *NS, EPS, s["work"].data_ptr(), s["work"].numel(), dt, stream))
    return out


def _own_muon(s):
    veda, lib, stream = _lib()
    c = s["case"]
    b, r, k = c["batch"], c["rows"], c["cols"]
    dt = veda.F32 if c["dtype"] == "f32" else veda.BF16
    if "work" not in s:
        s["work"] = torch.empty(lib.veda_muon_step_workspace(b, r, k, dt), dtype=torch.uint8,
                                device="cuda")
    low = s["lowp"]
    veda.check(lib.veda_muon_step(
        s["master"].data_ptr(), s["momentum"].data_ptr(), s["g"].data_ptr(),
        None if low is None else low.data_ptr(), b, r, k, r * k, LR, MOMENTUM, 1, DECAY,
        _update_scale(c), STEPS, *NS, EPS, None, 1.0, 1.0, 0, s["work"].data_ptr(),
        s["work"].numel(), stream))


def run(state):
    op = state["case"]["op"]
    if op == "loss":
        return _own_loss(state) if own else _plain_loss(state)
    if op == "orth":
        return _own_orth(state) if own else _plain_orth(state["g"]).to(state["g"].dtype)
    if own:
        _own_muon(state)
    else:
        _plain_muon(state)
    out = {"master": state["master"], "momentum": state["momentum"]}
    if state["lowp"] is not None:
        out["values"] = state["lowp"]
    return out


# ---- 64 bits -----------------------------------------------------------------------------------
def _exact_loss(case, seed):
    s = prepare(case, seed)
    w, t = s["w"].double(), s["t"]
    used = (t != IGNORE).nonzero()[:, 0]
    n = max(1, len(used))
    row = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(row)
    dx = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    for i in range(0, case["rows"], 512):
        x = s["x"][i:i + 512].double()
        z = torch.einsum("nd,vd->nv", x, w)
        lse[i:i + 512] = torch.logsumexp(z, 1)
        here = used[(used >= i) & (used < i + 512)]
        if not len(here):
            continue
        k = here - i
        row[here] = lse[here] - z[k, t[here]]
        if case["grads"]:
            q = torch.softmax(z[k], 1)
            q[torch.arange(len(k), device="cuda"), t[here]] -= 1.0
            dx[here] = torch.einsum("nv,vd->nd", q, w) / n
            dw += torch.einsum("nv,nd->vd", q, x[k]) / n
    out = {"loss": row.sum() / n, "row_loss": row, "lse": lse}
    if case["grads"]:
        out["dx"], out["dw"] = dx, dw
    return out


def _exact_orth(u):
    """The odd polynomial a s + b s^3 + c s^5 applied STEPS times through X <- (a + b S + c S^2) X."""
    x = u.double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT if flip else x
    x = x / (torch.linalg.matrix_norm(x)[:, None, None] + EPS)
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.einsum("bik,bjk->bij", x, x)
        x = torch.einsum("bij,bjk->bik", NS[0] * eye + NS[1] * gram
                         + NS[2] * torch.einsum("bij,bjk->bik", gram, gram), x)
    return x.mT if flip else x


def exact(case, seed):
    if case["op"] == "loss":
        return _exact_loss(case, seed)
    s = prepare(case, seed)
    if case["op"] == "orth":
        return _exact_orth(s["g"])
    g, w = s["g"].double(), s["master"].double()
    m = s["momentum"].double() * MOMENTUM + g
    step = 0.2 * max(case["rows"], case["cols"]) ** 0.5 * LR
    w = w * (1.0 - LR * DECAY) - step * _exact_orth(g + MOMENTUM * m)
    out = {"master": w, "momentum": m}
    if case["dtype"] == "bf16":
        out["values"] = w
    return out


# ---- work --------------------------------------------------------------------------------------
def _ns_flops(batch, rows, cols):
    """Products of STEPS iterations on the smaller side, the two symmetric ones counted by halves."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * batch * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "loss":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        flops, nbytes = 2.0 * n * v * d, e * (n * d + v * d) + 16 * n
        if case["grads"]:   # the two gradient products; the forward's logits are counted once
            flops, nbytes = 3 * flops, nbytes + e * (n * d + v * d)
        return {"bytes": nbytes, "flops": flops}
    size = case["batch"] * case["rows"] * case["cols"]
    flops = _ns_flops(case["batch"], case["rows"], case["cols"])
    if case["op"] == "orth":
        return {"bytes": 2 * e * size, "flops": flops}
    # gradient read, momentum and master read and written, bf16 weights written
    return {"bytes": size * (20 + (2 if case["dtype"] == "bf16" else 0)), "flops": flops}
