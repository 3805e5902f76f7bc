"""Measured operators of the training step's end: the norm in front of the head, the head's loss and a teacher's.

The kinds of case are

* ``norm``  ``layer_norm`` or ``rms_norm`` of T rows of width D, with a residual added first where ``residual``;
* ``ce``    ``linear_cross_entropy`` of T tokens of width D over a vocabulary of V;
* ``kd``    ``linear_distillation`` from a teacher's K top logits a token.

``train``: with the gradients.  ``order``: of the head's weight in memory, "dv" for [D, V] as it is written, "vd" for an
embedding table [V, D] that is passed transposed.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100
LN_EPS, RMS_EPS = 1e-5, 1e-6

# What the largest listed cases need bounds the drawn ones.
MAX_HEAD = 2.7e13  # flops of a loss and its gradients
MAX_NORM = 1.2e8   # elements


def _norm(T, D, rms=False, dtype="bf16", weight="bf16", residual=False, train=False):
    return dict(kind="norm", T=T, D=D, rms=rms, dtype=dtype, weight=weight, residual=residual, train=train)


def _ce(T, D, V, dtype="bf16", order="dv", z_loss=0.0, reduction="mean", train=True):
    return dict(kind="ce", T=T, D=D, V=V, dtype=dtype, order=order, z_loss=z_loss, reduction=reduction, train=train)


def _kd(T, D, V, K, dtype="bf16", order="dv", tau=1.0, reduction="mean", train=True):
    return dict(kind="kd", T=T, D=D, V=V, K=K, dtype=dtype, order=order, tau=tau, reduction=reduction, train=train)


def listed():
    return [
        # one user's next token on its way into a layer
        dict(_norm(1, 4096, rms=True, residual=True), name="norm_one_token"),
        # a training step of a dense layer's norm
        dict(_norm(8192, 4096, train=True), name="norm_train"),
        # a small experiment in 32 bits, at a width of no alignment
        dict(_norm(1000, 501, dtype="f32", weight="f32", train=True), name="norm_train_f32_odd"),
        # a training step of a wide model's norm behind its residual, weights in 32 bits, an odd number of tokens
        dict(_norm(16381, 7168, rms=True, weight="f32", residual=True, train=True), name="norm_train_wide"),
        # the answers of a multiple-choice question are scored, token by token
        dict(_ce(7, 2048, 32000, reduction="none", train=False), name="ce_score_few"),
        # a training step over an ordinary vocabulary
        dict(_ce(4096, 4096, 32000), name="ce_train"),
        # a training step of a small model whose vocabulary was not padded
        dict(_ce(1531, 704, 50257, z_loss=1e-4), name="ce_train_odd"),
        # a small experiment in 32 bits
        dict(_ce(1000, 512, 5003, dtype="f32", order="vd"), name="ce_train_f32"),
        # a training step over a large vocabulary, with the embedding table as the head
        dict(_ce(8192, 4096, 131072, order="vd", z_loss=1e-4), name="ce_train_large"),
        # the last few prompts of a distillation set
        dict(_kd(61, 1536, 32000, 8), name="kd_few"),
        # a distillation step from a large teacher, softened, with an odd number of tokens
        dict(_kd(4093, 2048, 131072, 64, tau=2.0), name="kd_train"),
        # the same of a small student: sizes of no alignment, the tokens weighted one by one
        dict(_kd(1531, 1001, 50257, 100, order="vd", reduction="none"), name="kd_train_odd"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(round(v / step) * step, math.ceil(lo / step) * step), hi // step * step))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "norm", "ce", "ce", "ce", "kd", "kd"])
        step = rng.choice([1, 8, 64, 64])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        if kind == "norm":
            c = _norm(_log(rng, 1, 32768), _log(rng, 64, 16384, step), rng.random() < 0.5, dtype,
                      rng.choice([dtype, "f32"]), rng.random() < 0.5, rng.random() < 0.6)
            if c["T"] * c["D"] <= MAX_NORM:
                return c
            continue
        T, D = _log(rng, 1, 8192), _log(rng, 64, 4096, step)
        V = _log(rng, 1000, 131072, rng.choice([1, 64, 256]))
        order, reduction = rng.choice(["dv", "vd"]), rng.choice(["mean", "none"])
        train = rng.random() < 0.75
        if kind == "ce":
            c = _ce(T, D, V, dtype, order, rng.choice([0.0, 1e-4]), reduction, train)
        else:
            c = _kd(T, D, V, _log(rng, 1, 256), dtype, order, rng.choice([1.0, 2.0, 0.7]), reduction, train)
        if work(c)["flops"] <= MAX_HEAD / (16 if dtype == "f32" else 1):
            return c


def work(case):
    c = case
    s = 4 if c["dtype"] == "f32" else 2
    T, D = c["T"], c["D"]
    if c["kind"] == "norm":
        tensors = 4 if c["residual"] else 2  # x (and residual) read, y (and h) written
        moved = T * D * tensors * s
        if c["train"]:  # h again and dy (and dh) read, dx written
            moved += T * D * (4 if c["residual"] else 3) * s
        params = D * (1 if c["rms"] else 2) * (4 if c["weight"] == "f32" else 2)
        return {"bytes": moved + params * (3 if c["train"] else 1), "flops": T * D * (20 if c["train"] else 8)}
    V = c["V"]
    moved = s * (T * D + D * V) * (2 if c["train"] else 1) + 4 * T  # operands read, gradients written
    moved += 8 * T if c["kind"] == "ce" else 8 * T * c["K"]
    return {"bytes": moved, "flops": 2 * T * D * V * (3 if c["train"] else 1)}


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = DTYPES[c["dtype"]]
    T, D = c["T"], c["D"]

    def normal(*shape, std=1.0, mean=0.0, dtype=t):
        return (torch.randn(shape, device=DEV, generator=g) * std + mean).to(dtype)

    s = {"case": c}
    if c["kind"] == "norm":
        # a residual stream: sizes differ from token to token and from feature to feature, a few features are far off
        rows = torch.exp(0.5 * torch.randn((T, 1), device=DEV, generator=g))
        cols = torch.exp(0.7 * torch.randn((1, D), device=DEV, generator=g))
        s["x"] = (torch.randn((T, D), device=DEV, generator=g) * rows * cols + 0.2).to(t)
        s["residual"] = normal(T, D, std=2.0) if c["residual"] else None
        w = DTYPES[c["weight"]]
        s["weight"] = normal(D, std=0.2, mean=1.0, dtype=w)
        s["bias"] = None if c["rms"] else normal(D, std=0.2, dtype=w)
        if c["train"]:
            s["dy"] = normal(T, D)
            s["dh"] = normal(T, D) if c["residual"] else None
            s["leaves"] = [v.requires_grad_(True) for v in (s["x"], s["residual"], s["weight"], s["bias"]) if v is not None]
        return s
    V = c["V"]
    # logits of size 1.5, the right token's raised so that it has a fair share of the probability
    table = normal(V, D, std=1.5 * D ** -0.5)
    likely = (torch.exp(torch.rand(T, device=DEV, generator=g) * math.log(V)) - 1).long().clamp(0, V - 1)
    x = (torch.randn((T, D), device=DEV, generator=g) + 5.0 * table[likely].float()).to(t)
    s["weight"] = table.t() if c["order"] == "vd" else table.t().contiguous()
    s["x"] = x
    if c["kind"] == "ce":
        right = torch.rand(T, device=DEV, generator=g) < 0.8
        other = torch.randint(0, V, (T,), device=DEV, generator=g)
        y = torch.where(right, likely, other)
        s["targets"] = torch.where(torch.rand(T, device=DEV, generator=g) < (0.05 if T > 32 else 0.0), IGNORE, y)
    else:
        # a teacher's logits, falling from the first; entries of a row lie close together or far apart, all of them
        # distinct; some rows hold fewer than K entries, some none (padding)
        K = c["K"]
        k = torch.arange(K, device=DEV)
        far = torch.exp(torch.rand((T, 1), device=DEV, generator=g) * math.log(max(V // K, 1))).long().clamp(1, max(V // K, 1))
        idx = (likely[:, None] + k * far) % V
        live = (torch.rand((T, 1), device=DEV, generator=g) * K * 4 + 1).long()
        pad = torch.rand((T, 1), device=DEV, generator=g) < (0.05 if T > 32 else 0.0)
        s["indices"] = torch.where((k < live) & ~pad, idx, -1).to(torch.int32)
        s["teacher"] = 9.0 - 1.5 * torch.log1p(k.float()) + 0.3 * torch.randn((T, K), device=DEV, generator=g)
    if c["train"]:
        s["g"] = torch.rand(T, device=DEV, generator=g) / T if c["reduction"] == "none" else None
        s["leaves"] = [s["x"].requires_grad_(True), s["weight"].requires_grad_(True)]
    return s


def _plain_norm(s):
    c = s["case"]
    t = s["x"].dtype
    with torch.no_grad():
        h = s["x"]
        if c["residual"]:
            h = (h.float() + s["residual"].float()).to(t)
        v, w = h.float(), s["weight"].float()
        if c["rms"]:
            d = v
            rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + RMS_EPS)
        else:
            d = v - v.mean(-1, keepdim=True)
            rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + LN_EPS)
        n = d * rstd
        y = n * w if c["rms"] else n * w + s["bias"].float()
        out = [y.to(t)] + ([h] if c["residual"] else [])
        if not c["train"]:
            return out
        dy = s["dy"].float()
        u = dy * w
        dx = u - n * (u * n).mean(-1, keepdim=True)
        if not c["rms"]:
            dx = dx - u.mean(-1, keepdim=True)
        dx = dx * rstd
        if c["residual"]:
            dx = dx + s["dh"].float()
        dx = dx.to(t)
        out += [dx, dx] if c["residual"] else [dx]
        out.append((dy * n).sum(0).to(s["weight"].dtype))
        if not c["rms"]:
            out.append(dy.sum(0).to(s["weight"].dtype))
        return out


def _plain_head(s):
    c = s["case"]
    T, t = c["T"], s["x"].dtype
    with torch.no_grad():
        x, w = s["x"].float(), s["weight"].float()
        z = x @ w
        if c["kind"] == "ce":
            k = 1.0
            live = s["targets"] != IGNORE
            at = torch.where(live, s["targets"], 0)[:, None].long()
            share = live[:, None].float()
            const = torch.zeros(T, device=z.device)
        else:
            k = 1.0 / c["tau"]
            on = s["indices"] >= 0
            live = on.any(1)
            at = torch.where(on, s["indices"], 0).long()
            v = torch.where(on, s["teacher"] * k, -math.inf)
            v = torch.where(live[:, None], v, 0.0)
            e = torch.exp(v - v.amax(1, keepdim=True)) * on
            share = e / e.sum(1, keepdim=True).clamp(min=1e-30)
            const = torch.where(share > 0, share * torch.log(share.clamp(min=1e-37)), 0.0).sum(1)
        z *= k
        m = z.amax(1, keepdim=True)
        chosen = z.gather(1, at)
        z -= m
        z.exp_()
        total = z.sum(1, keepdim=True)
        lse = (m + torch.log(total))[:, 0]
        loss = torch.where(live, const + lse - (share * chosen).sum(1), 0.0)
        slope = 1.0
        if c["kind"] == "ce":
            loss = torch.where(live, loss + c["z_loss"] * lse * lse, 0.0)
            slope = 1 + 2 * c["z_loss"] * lse
        else:
            loss = loss * c["tau"] ** 2
        count = live.sum().clamp(min=1)
        out = [loss if c["reduction"] == "none" else loss.sum() / count]
        if not c["train"]:
            return out
        g = s["g"] if c["reduction"] == "none" else 1.0 / count
        g = torch.where(live, g, 0.0) * (c["tau"] if c["kind"] == "kd" else 1.0)
        z *= (g * slope)[:, None] / total
        z.scatter_add_(1, at, -g[:, None] * share)
        out += [(z @ w.t()).to(t), (x.t() @ z).to(t)]
        return out


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _plain_norm(s) if c["kind"] == "norm" else _plain_head(s)
    if c["kind"] == "norm":
        from mintext_amd.kernels import layer_norm, rms_norm
        if c["rms"]:
            out = rms_norm(s["x"], s["weight"], eps=RMS_EPS, residual=s["residual"])
        else:
            out = layer_norm(s["x"], s["weight"], s["bias"], eps=LN_EPS, residual=s["residual"])
        out = list(out) if c["residual"] else [out]
        if c["train"]:
            out += torch.autograd.grad(out, s["leaves"], [s["dy"]] + ([s["dh"]] if c["residual"] else []))
        return out
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation
    if c["kind"] == "ce":
        loss = linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, z_loss=c["z_loss"],
                                    reduction=c["reduction"])
    else:
        loss = linear_distillation(s["x"], s["weight"], s["indices"], s["teacher"], temperature=c["tau"],
                                   reduction=c["reduction"])
    return [loss] + (list(torch.autograd.grad(loss, s["leaves"], s["g"])) if c["train"] else [])


def _exact_norm(c, s):
    v = [s[k] if s[k] is None else s[k].detach().double().requires_grad_(c["train"])
         for k in ("x", "residual", "weight", "bias")]
    x, r, w, b = v
    if r is None:
        h = x
    else:
        # the sum as the operator hands it on, in the operands' type; its rounding has no gradient of its own
        h = x + r
        h = h + (h.detach().float().to(DTYPES[c["dtype"]]).double() - h.detach())
    if c["rms"]:
        y = h * (h.pow(2).mean(-1, keepdim=True) + RMS_EPS).rsqrt() * w
    else:
        var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
        y = (h - mean) * (var + LN_EPS).rsqrt() * w + b
    out = [y] if r is None else [y, h]
    res = [o.detach() for o in out]
    if c["train"]:
        leaves = [p for p in v if p is not None]
        res += torch.autograd.grad(out, leaves, [s["dy"].double()] + ([s["dh"].double()] if r is not None else []))
    return res


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "norm":
        return _exact_norm(c, s)
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    z = torch.mm(x, w)
    if c["kind"] == "kd":
        z /= c["tau"]
    lse = torch.empty(c["T"], dtype=torch.float64, device=DEV)
    for i in range(0, c["T"], 1024):
        lse[i:i + 1024] = torch.logsumexp(z[i:i + 1024], 1)
    if c["kind"] == "ce":
        live = s["targets"] != IGNORE
        rows = live.nonzero()[:, 0]
        cols, p = s["targets"][rows].long(), torch.ones(len(rows), dtype=torch.float64, device=DEV)
        loss = torch.where(live, lse + c["z_loss"] * lse ** 2, 0.0)
        loss.index_put_((rows,), -z[rows, cols], accumulate=True)
        front = 1 + 2 * c["z_loss"] * lse
        unit = 1.0
    else:
        live = (s["indices"] >= 0).any(1)
        rows, k = (s["indices"] >= 0).nonzero(as_tuple=True)
        cols = s["indices"][rows, k].long()
        e = torch.exp(s["teacher"][rows, k].double() / c["tau"])
        p = e / torch.zeros_like(lse).index_add_(0, rows, e)[rows]
        loss = torch.zeros_like(lse).index_add_(0, rows, p * (torch.log(p) - z[rows, cols] + lse[rows])) * c["tau"] ** 2
        front = torch.ones_like(lse)
        unit = c["tau"]
    n = max(int(live.sum()), 1)
    out = [loss if c["reduction"] == "none" else loss.sum() / n]
    if c["train"]:
        g = unit * live.double() * (s["g"].double() if c["reduction"] == "none" else 1.0 / n)
        z.sub_(lse[:, None]).exp_().mul_((g * front)[:, None])
        z.index_put_((rows, cols), -g[rows] * p, accumulate=True)
        out += [torch.mm(z, w.t()), torch.mm(x.t(), z)]
    return out
