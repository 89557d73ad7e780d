"""The workloads of the MXFP4 operators and the distillation loss, with their plain forms.

Operators: MXFP4 quantisation (E2M1 elements, one power-of-two scale per 32), the MXFP4 linear
layer and its backward pass, the gated (SwiGLU) feed-forward block and its backward pass, and the
distillation loss from a teacher's top logits with its gradient.

``run`` computes an operator in elementary torch operations in fp32 (``own`` false) or makes the
calls a user makes of the framework (``own`` true); ``exact`` computes it in fp64 from the
operator's definition, written apart from the plain form.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # the activations of a training step's linear layer, quantised along both axes for its three products
        {"name": "quantise-train-8192x4096", "op": "quantise", "rows": 8192, "cols": 4096, "dtype": "bf16", "dual": True},
        # a handful of fp32 rows with an odd width: latency and a short last block
        {"name": "quantise-few-17x4095", "op": "quantise", "rows": 17, "cols": 4095, "dtype": "f32", "dual": False},
        # one token through a gate/up projection whose weights are kept in 4 bits
        {"name": "linear-token-1x4096x22016", "op": "linear", "tokens": 1, "inp": 4096, "out": 22016, "dtype": "bf16", "bias": False},
        # a small decoding batch through a down projection, fp16 activations, a bias
        {"name": "linear-batch-33x11008x4096", "op": "linear", "tokens": 33, "inp": 11008, "out": 4096, "dtype": "f16", "bias": True},
        # a prompt of 4000 tokens through a query/key/value projection
        {"name": "linear-prompt-4000x4096x12288", "op": "linear", "tokens": 4000, "inp": 4096, "out": 12288, "dtype": "bf16", "bias": False},
        # a training step (forward, all gradients) of the decoder's up projection
        {"name": "linear-train-8192x2048x8192", "op": "linear_train", "tokens": 8192, "inp": 2048, "out": 8192, "dtype": "bf16", "bias": True},
        # one token through the whole gated block
        {"name": "gated-token-1x4096x11008", "op": "gated", "tokens": 1, "d": 4096, "f": 11008, "dtype": "bf16"},
        # a prompt of odd length through the gated block
        {"name": "gated-prompt-1777x4096x11008", "op": "gated", "tokens": 1777, "d": 4096, "f": 11008, "dtype": "bf16"},
        # a training step of the gated block
        {"name": "gated-train-8192x4096x11008", "op": "gated_train", "tokens": 8192, "d": 4096, "f": 11008, "dtype": "bf16"},
        # held-out evaluation of a few positions: the loss of each, no gradient
        {"name": "distil-eval-64x32000", "op": "distil", "rows": 64, "vocab": 32000, "top": 20, "dtype": "f32",
         "temperature": 1.0, "alpha": 1.0, "labels": False, "tail": False, "grad": False},
        # one micro-batch (8 sequences of 2048) of the decoder, hard labels and the teacher's top 64
        {"name": "distil-train-16384x32000", "op": "distil", "rows": 16384, "vocab": 32000, "top": 64, "dtype": "bf16",
         "temperature": 2.0, "alpha": 0.5, "labels": True, "tail": False, "grad": True},
        # a long odd vocabulary, the teacher's true probabilities with a bucket for the rest
        {"name": "distil-tail-1500x131071", "op": "distil", "rows": 1500, "vocab": 131071, "top": 100, "dtype": "bf16",
         "temperature": 1.0, "alpha": 1.0, "labels": False, "tail": True, "grad": True},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["quantise", "linear", "linear_train", "gated", "gated_train", "distil"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantise":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "cols": _log_int(rng, 16, 4096), "dtype": dtype,
                "dual": rng.random() < 0.5}
    if op == "linear":
        return {"op": op, "tokens": _log_int(rng, 1, 4000), "inp": _log_int(rng, 64, 4096), "out": _log_int(rng, 64, 12288),
                "dtype": dtype, "bias": rng.random() < 0.5}
    if op == "linear_train":
        return {"op": op, "tokens": _log_int(rng, 16, 8192), "inp": _log_int(rng, 64, 2048), "out": _log_int(rng, 64, 8192),
                "dtype": "bf16", "bias": rng.random() < 0.5}
    if op == "gated":
        return {"op": op, "tokens": _log_int(rng, 1, 1777), "d": _log_int(rng, 64, 4096),
                "f": 32 * _log_int(rng, 2, 344), "dtype": dtype}
    if op == "gated_train":
        return {"op": op, "tokens": _log_int(rng, 16, 8192), "d": _log_int(rng, 64, 4096),
                "f": 32 * _log_int(rng, 2, 344), "dtype": "bf16"}
    vocab = _log_int(rng, 1000, 131071)
    return {"op": op, "rows": _log_int(rng, 1, max(1, min(16384, 16384 * 32000 // (2 * vocab)))), "vocab": vocab,
            "top": _log_int(rng, 1, 128), "dtype": dtype, "temperature": rng.choice([1.0, 2.0, 0.7, 4.0]),
            "alpha": rng.choice([1.0, 0.5, 0.9]), "labels": rng.random() < 0.5, "tail": rng.random() < 0.4,
            "grad": rng.random() < 0.7}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _activations(rows: int, cols: int, gen, dtype) -> torch.Tensor:
    """Rows of activations: normal, with a few channels much larger than the rest."""
    x = torch.randn(rows, cols, device=DEV, generator=gen)
    big = (torch.rand(cols, device=DEV, generator=gen) < 0.004).float() * 15.0 + 1.0
    return (x * big).to(dtype)


def _inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    op = case["op"]
    dt = DTYPES[case["dtype"]]
    if op == "quantise":
        return {"x": _activations(case["rows"], case["cols"], g, dt)}
    if op in ("linear", "linear_train"):
        t, k, o = case["tokens"], case["inp"], case["out"]
        s = {"x": _activations(t, k, g, dt), "w": (torch.randn(o, k, device=DEV, generator=g) * 0.02).to(torch.bfloat16)}
        s["b"] = (torch.randn(o, device=DEV, generator=g) * 0.1) if case["bias"] else None
        if op == "linear_train":
            s["dy"] = (torch.randn(t, o, device=DEV, generator=g) * 1e-3).to(torch.bfloat16)
        return s
    if op in ("gated", "gated_train"):
        t, d, f = case["tokens"], case["d"], case["f"]
        s = {"x": _activations(t, d, g, dt),
             "wgu": (torch.randn(2 * f, d, device=DEV, generator=g) * 0.02).to(torch.bfloat16),
             "wd": (torch.randn(d, f, device=DEV, generator=g) * 0.02).to(torch.bfloat16)}
        if op == "gated_train":
            s["dy"] = (torch.randn(t, d, device=DEV, generator=g) * 1e-3).to(torch.bfloat16)
        return s
    n, v, k = case["rows"], case["vocab"], min(case["top"], case["vocab"])
    logits = torch.empty(n, v, device=DEV, dtype=dt)
    ids = torch.empty(n, k, device=DEV, dtype=torch.int64)
    tl = torch.empty(n, k, device=DEV, dtype=torch.float32)
    lse = torch.empty(n, device=DEV, dtype=torch.float32)
    for i in range(0, n, 2048):  # the teacher agrees with the student up to noise
        z = torch.randn(min(2048, n - i), v, device=DEV, generator=g) * 2.5
        logits[i:i + 2048] = z.to(dt)
        z += torch.randn(z.shape, device=DEV, generator=g) * 0.7
        top = torch.topk(z, k, dim=1)
        ids[i:i + 2048], tl[i:i + 2048] = top.indices, top.values
        lse[i:i + 2048] = torch.logsumexp(z / case["temperature"], dim=1)
    # some rows keep fewer entries than others (padded with -1)
    keep = torch.randint(1, k + 1, (n, 1), device=DEV, generator=g)
    full = torch.rand(n, 1, device=DEV, generator=g) < 0.8
    ids = torch.where(full | (torch.arange(k, device=DEV)[None] < keep), ids, torch.full_like(ids, -1))
    s = {"logits": logits, "ids": ids, "tl": tl, "lse": lse if case["tail"] else None, "labels": None}
    if case["labels"]:
        lab = torch.randint(0, v, (n,), device=DEV, generator=g)
        drop = torch.rand(n, device=DEV, generator=g) < 0.1  # padding positions
        s["labels"] = torch.where(drop, torch.full_like(lab, -100), lab)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    if op in ("linear", "gated"):  # inference keeps its weights in 4 bits
        names = ("w",) if op == "linear" else ("wgu", "wd")
        if own:
            from firefly_b200 import quantize_fp_to_mxfp4
            for n in names:
                s[n] = quantize_fp_to_mxfp4(s[n])
        else:
            for n in names:
                s[n] = _mx(s[n])
    elif own:
        for n in {"linear_train": ("x", "w", "b"), "gated_train": ("x", "wgu", "wd"), "distil": ("logits",)}.get(op, ()):
            if s[n] is not None and (op != "distil" or case["grad"]):
                s[n].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# plain forms (fp32)
# ---------------------------------------------------------------------------
def _mx(x: torch.Tensor) -> torch.Tensor:
    """The values that the MXFP4 codes of x stand for (blocks of 32 along the last axis), fp32."""
    x = x.float()
    r, c = x.shape
    pad = (-c) % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros(r, pad)], dim=1)
    xb = x.view(r, -1, BLOCK)
    amax = xb.abs().amax(dim=2, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, torch.full_like(amax, -127, dtype=torch.int32)).clamp(min=-127)
    a = torch.ldexp(xb.abs(), -e).clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.ldexp(torch.round(a / step) * step, e) * torch.sign(xb)
    return q.view(r, -1)[:, :c]


def _bf(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.bfloat16)


def _plain_quantise(s):
    # the codes' values have at most two significant bits: bf16 holds them exactly
    out = [_bf(_mx(s["x"]))]
    if s["case"]["dual"]:
        out.append(_bf(_mx(s["x"].t().contiguous())))
    return out


def _plain_linear(s):
    y = _mx(s["x"]) @ s["w"].t()
    return _bf(y if s["b"] is None else y + s["b"])


def _plain_linear_train(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    y = _mx(x) @ _mx(w).t()
    if s["b"] is not None:
        y = y + s["b"]
    out = {"y": _bf(y), "dx": _bf(_mx(dy) @ _mx(w.t().contiguous()).t()),
           "dw": _bf(_mx(dy.t().contiguous()) @ _mx(x.t().contiguous()).t())}
    if s["b"] is not None:
        out["db"] = dy.float().sum(0)
    return out


def _plain_gated_fwd(x, wgu, wd):
    f = wd.shape[1]
    gu = _bf(_mx(x) @ wgu.t())  # the activations between the products are held in bf16
    g, u = gu[:, :f].float(), gu[:, f:].float()
    h = _bf(g / (1 + torch.exp(-g)) * u)
    return g, u, h, _bf(_mx(h) @ wd.t())


def _plain_gated_train(s):
    x, wgu, wd, dy = s["x"], s["wgu"], s["wd"], s["dy"]
    g, u, h, y = _plain_gated_fwd(x, _mx(wgu), _mx(wd))
    dh = _bf(_mx(dy) @ _mx(wd.t().contiguous()).t()).float()
    sig = 1 / (1 + torch.exp(-g))
    dgu = _bf(torch.cat([dh * u * sig * (1 + g * (1 - sig)), dh * g * sig], dim=1))
    dgut = dgu.t().contiguous()
    return {"y": y, "dx": _bf(_mx(dgu) @ _mx(wgu.t().contiguous()).t()),
            "dwgu": _bf(_mx(dgut) @ _mx(x.t().contiguous()).t()),
            "dwd": _bf(_mx(dy.t().contiguous()) @ _mx(h.t().contiguous()).t())}


def _plain_distil(s):
    c = s["case"]
    T, alpha = c["temperature"], c["alpha"]
    ids, labels = s["ids"], s["labels"]
    z = s["logits"].float()
    n, v = z.shape
    on = ids >= 0
    at = ids.clamp(min=0)
    zt = z / T
    m = zt.amax(1, keepdim=True)
    ex = torch.exp(zt - m)
    total = ex.sum(1, keepdim=True)
    lse = m + torch.log(total)
    t = torch.where(on, s["tl"] / T, torch.full_like(s["tl"], -math.inf))
    if s["lse"] is not None:
        logp = t - s["lse"][:, None]
    else:
        tm = t.amax(1, keepdim=True)
        logp = t - (tm + torch.log(torch.exp(t - tm).sum(1, keepdim=True)))
    p = torch.where(on, torch.exp(logp), torch.zeros_like(logp))
    kd = torch.where(on & (p > 0), p * (logp - (zt.gather(1, at) - lse)), torch.zeros_like(p)).sum(1)
    counted = labels != -100 if labels is not None else on.any(1)
    scale = torch.ones_like(lse)  # the factor of q off the teacher's ids
    if s["lse"] is not None:
        has = on.any(1)
        mark = torch.zeros(n, v, dtype=torch.bool, device=z.device)
        rr = torch.arange(n, device=z.device)[:, None].expand_as(at)[on]
        mark[rr, at[on]] = True
        qt = torch.where(mark, torch.zeros_like(ex), ex).sum(1) / total[:, 0]
        pt = (1 - p.sum(1)).clamp(min=0)
        kd = kd + torch.where(has & (pt > 0), pt * (torch.log(pt) - torch.log(qt)), torch.zeros_like(pt))
        scale = torch.where(has & (qt > 0), 1 - pt / qt, torch.ones_like(pt))[:, None]
    kd = kd * T * T
    loss = alpha * kd
    if labels is not None:
        m1 = z.amax(1, keepdim=True)
        e1 = torch.exp(z - m1)
        tot1 = e1.sum(1, keepdim=True)
        lab = labels.clamp(min=0)[:, None]
        loss = loss + (1 - alpha) * (m1 + torch.log(tot1) - z.gather(1, lab))[:, 0]
    loss = torch.where(counted, loss, torch.zeros_like(loss))
    if not c["grad"]:
        return [loss]
    q = ex / total
    gz = q * scale if s["lse"] is None else torch.where(mark, q, q * scale)
    gz.scatter_add_(1, at, -p)
    gz = torch.where(on.any(1)[:, None], gz, torch.zeros_like(gz)) * (alpha * T)
    if labels is not None:
        g1 = e1 / tot1
        g1.scatter_add_(1, lab, torch.full_like(m1, -1.0))
        gz = gz + (1 - alpha) * g1
    cnt = counted.sum().clamp(min=1)
    grad = torch.where(counted[:, None], gz, torch.zeros_like(gz)) / cnt
    return [loss.sum() / cnt, grad.to(s["logits"].dtype)]


def _plain(s):
    op = s["case"]["op"]
    if op == "quantise":
        return _plain_quantise(s)
    if op == "linear":
        return _plain_linear(s)
    if op == "linear_train":
        return _plain_linear_train(s)
    if op == "gated":
        return _plain_gated_fwd(s["x"], s["wgu"], s["wd"])[3]
    if op == "gated_train":
        return _plain_gated_train(s)
    return _plain_distil(s)


# ---------------------------------------------------------------------------
# the framework's operators, as a user's program calls them
# ---------------------------------------------------------------------------
def _own(s):
    import firefly_b200 as ff

    c = s["case"]
    op = c["op"]
    if op == "quantise":
        if c["dual"]:
            return [q.dequantize(torch.bfloat16) for q in ff.quantize_fp_to_mxfp4_dual(s["x"])]
        return [ff.quantize_fp_to_mxfp4(s["x"]).dequantize(torch.bfloat16)]
    if op == "linear":
        return ff.mxfp4_linear(s["x"], s["w"], s["b"])
    if op == "linear_train":
        y = ff.mxfp4_linear(s["x"], s["w"], s["b"])
        leaves = [s["x"], s["w"]] + ([s["b"]] if s["b"] is not None else [])
        grads = torch.autograd.grad(y, leaves, s["dy"])
        return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *grads)))
    if op == "gated":
        return ff.mxfp4_swiglu(s["x"], s["wgu"], s["wd"])
    if op == "gated_train":
        y = ff.mxfp4_swiglu(s["x"], s["wgu"], s["wd"])
        grads = torch.autograd.grad(y, [s["x"], s["wgu"], s["wd"]], s["dy"])
        return dict(zip(("y", "dx", "dwgu", "dwd"), (y.detach(), *grads)))
    loss = ff.distillation_loss(s["logits"], s["ids"], s["tl"], labels=s["labels"], teacher_lse=s["lse"],
                                temperature=c["temperature"], alpha=c["alpha"],
                                reduction="mean" if c["grad"] else "none")
    if not c["grad"]:
        return [loss]
    return [loss.detach(), torch.autograd.grad(loss, s["logits"])[0]]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    op = case["op"]
    b = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    packed = 0.5 + 1 / BLOCK  # bytes of a value held in the format
    if op == "quantise":
        n = case["rows"] * case["cols"]
        # the packed form is written and read back, its values written in bf16
        return {"bytes": n * b + (2 if case["dual"] else 1) * n * (2 * packed + 2), "flops": 0}
    if op in ("linear", "linear_train"):
        t, k, o = case["tokens"], case["inp"], case["out"]
        if op == "linear":
            return {"bytes": t * k * b + o * k * packed + t * o * 2 + (4 * o if case["bias"] else 0), "flops": 2 * t * k * o}
        return {"bytes": 2 * (t * k * b + o * k * 2) + 2 * t * o * 2 + (8 * o if case["bias"] else 0), "flops": 6 * t * k * o}
    if op in ("gated", "gated_train"):
        t, d, f = case["tokens"], case["d"], case["f"]
        if op == "gated":
            return {"bytes": t * d * (b + 2) + 3 * d * f * packed, "flops": 6 * t * d * f}
        return {"bytes": 4 * t * d * 2 + 2 * 3 * d * f * 2, "flops": 18 * t * d * f}
    n, v, k = case["rows"], case["vocab"], min(case["top"], case["vocab"])
    nbytes = n * v * b * (2 if case["grad"] else 1) + n * k * 12 + n * (8 if case["labels"] else 0) + n * (4 if case["tail"] else 0)
    return {"bytes": nbytes, "flops": 6 * n * v}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _mx64(x: torch.Tensor) -> torch.Tensor:
    """MXFP4 values by counting the rounding thresholds below |x| / scale (ties to the even code)."""
    x = x.double()
    r, c = x.shape
    xp = torch.nn.functional.pad(x, (0, (-c) % BLOCK)).reshape(r, -1, BLOCK)
    amax = xp.abs().amax(2, keepdim=True)
    lg = torch.floor(torch.log2(amax.clamp(min=1e-300)))
    lg = torch.where(torch.exp2(lg + 1) <= amax, lg + 1, torch.where(torch.exp2(lg) > amax, lg - 1, lg))
    scale = torch.exp2((lg - 2).clamp(min=-127))
    a = xp.abs() / scale
    code = torch.zeros_like(a, dtype=torch.int64)
    for t in (0.25, 1.25, 2.5, 5.0):
        code += a > t
    for t in (0.75, 1.75, 3.5):
        code += a >= t
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (torch.copysign(levels[code], xp) * scale).reshape(r, -1)[:, :c]


def _prod64(a, b):
    """a @ b.T in fp64, the columns of the result in slices."""
    return torch.cat([a @ b[i:i + 4096].t() for i in range(0, b.shape[0], 4096)], dim=1)


def _half(x):
    return x.to(torch.bfloat16).double()


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantise":
        out = [_mx64(s["x"])]
        return out + [_mx64(s["x"].t())] if case["dual"] else out
    if op in ("linear", "linear_train"):
        y = _prod64(_mx64(s["x"]), _mx64(s["w"]))
        if s["b"] is not None:
            y = y + s["b"].double()
        if op == "linear":
            return y
        out = {"y": y, "dx": _prod64(_mx64(s["dy"]), _mx64(s["w"].t())),
               "dw": _prod64(_mx64(s["dy"].t()), _mx64(s["x"].t()))}
        if s["b"] is not None:
            out["db"] = s["dy"].double().sum(0)
        return out
    if op in ("gated", "gated_train"):
        f = case["f"]
        gu = _half(_prod64(_mx64(s["x"]), _mx64(s["wgu"])))
        g, u = gu[:, :f], gu[:, f:]
        h = _half(g * torch.sigmoid(g) * u)
        y = _prod64(_mx64(h), _mx64(s["wd"]))
        if op == "gated":
            return y
        dh = _half(_prod64(_mx64(s["dy"]), _mx64(s["wd"].t())))
        sg = torch.sigmoid(g)
        dgu = _half(torch.cat([dh * u * (sg + g * sg * (1 - sg)), dh * (g * sg)], 1))
        return {"y": y, "dx": _prod64(_mx64(dgu), _mx64(s["wgu"].t())),
                "dwgu": _prod64(_mx64(dgu.t()), _mx64(s["x"].t())),
                "dwd": _prod64(_mx64(s["dy"].t()), _mx64(h.t()))}
    T, alpha = case["temperature"], case["alpha"]
    n = case["rows"]
    losses, grads, counts = [], [], []
    for i in range(0, n, 1024):
        z = s["logits"][i:i + 1024].double().detach().requires_grad_(case["grad"])
        ids = s["ids"][i:i + 1024]
        on = ids >= 0
        at = torch.where(on, ids, torch.zeros_like(ids))
        has = on.any(1)
        t = (s["tl"][i:i + 1024].double() / T).masked_fill(~on, -math.inf)
        logq = torch.log_softmax(z / T, 1)
        logp = t - (s["lse"][i:i + 1024].double()[:, None] if s["lse"] is not None else torch.logsumexp(t, 1, keepdim=True))
        p = torch.exp(logp).masked_fill(~on, 0.0)
        row = (p * (logp.masked_fill(~on, 0.0) - logq.gather(1, at))).masked_fill(~on, 0.0).sum(1)
        if s["lse"] is not None:
            hit = torch.zeros(z.shape, dtype=torch.int32, device=z.device).scatter_add_(1, at, on.int()) > 0
            tail = torch.logsumexp(logq.masked_fill(hit, -math.inf), 1)
            pt = (1 - p.sum(1)).clamp(min=0)
            row = row + torch.where(has & (pt > 0), pt * (torch.log(pt) - tail), torch.zeros_like(pt))
        row = alpha * T * T * torch.where(has, row, torch.zeros_like(row))
        counted = has
        if s["labels"] is not None:
            lab = s["labels"][i:i + 1024]
            counted = lab != -100
            ce = -torch.log_softmax(z, 1).gather(1, lab.clamp(min=0)[:, None])[:, 0]
            row = row + (1 - alpha) * ce
        row = torch.where(counted, row, torch.zeros_like(row))
        if case["grad"]:
            grads.append(torch.autograd.grad(row.sum(), z)[0].float())
        losses.append(row.detach())
        counts.append(counted.sum())
    loss = torch.cat(losses)
    if not case["grad"]:
        return [loss]
    cnt = int(torch.stack(counts).sum().clamp(min=1))
    return [loss.sum() / cnt, torch.cat([gr / cnt for gr in grads])]
