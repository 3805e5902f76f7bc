"""Measured operators: the dense product with its epilogue, and the orthogonalised update of the weights.

The kinds of case are

* ``linear``   ``act(x @ w + bias) + residual`` of T rows, K x N weights; ``train``: with its gradients;
* ``ns``       ``newton_schulz`` of a stack of E matrices of M x N;
* ``muon``     ``muon_update`` of such a stack: momentum, orthogonalisation, weight decay and update.

``rank`` is the number of tokens whose outer products made a matrix's gradient, which bounds its rank.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
A, B, C = 3.4445, -4.7750, 2.0315  # the quintic's coefficients
STEPS, EPS = 5, 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.1
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")

# What the largest listed cases need bounds the drawn ones.
MAX_LINEAR = 9.0e11  # flops of a product and its gradients
MAX_STACK = 4.0e12   # flops of an orthogonalisation
MAX_ELEMENTS = 2.5e8


def _linear(T, K, N, act="none", dtype="bf16", bias=True, residual=False, train=False):
    return dict(kind="linear", T=T, K=K, N=N, act=act, dtype=dtype, bias=bias, residual=residual, train=train)


def _stack(kind, E, M, N, rank, dtype="bf16"):
    return dict(kind=kind, E=E, M=M, N=N, rank=rank, dtype=dtype)


def listed():
    return [
        # one user's next token through a wide projection: its weights are read once
        dict(_linear(1, 4096, 14336, "silu"), name="linear_one_token"),
        # a serving batch's next tokens, projected back onto the residual stream
        dict(_linear(61, 7168, 2048, residual=True), name="linear_decode_batch"),
        # a short prompt, widths that are no multiple of 128
        dict(_linear(1531, 1536, 704, "gelu", residual=True), name="linear_prompt"),
        # a long prompt batch through a dense MLP's first product
        dict(_linear(8192, 4096, 14336, "gelu_tanh"), name="linear_prefill"),
        # a training step of a dense projection with an odd number of tokens
        dict(_linear(4093, 2048, 7168, "silu", residual=True, train=True), name="linear_train"),
        # a small experiment in 32 bits, at widths of no alignment
        dict(_linear(1000, 501, 250, "gelu", dtype="f32", residual=True, train=True), name="linear_train_f32_odd"),
        # the experts of the smallest model that is run at all, in 32 bits
        dict(_stack("ns", 8, 128, 512, 64, "f32"), name="ns_tiny_f32"),
        # a few matrices of odd sizes, taller than wide
        dict(_stack("ns", 3, 1001, 333, 500), name="ns_odd"),
        # the gate projections of 128 narrow experts
        dict(_stack("ns", 128, 2048, 768, 1024), name="ns_experts"),
        # the step of one dense projection
        dict(_stack("muon", 1, 7168, 2048, 4096), name="muon_dense"),
        # the step of a small experiment's experts, weights in 32 bits
        dict(_stack("muon", 16, 512, 384, 250, "f32"), name="muon_experts_f32"),
        # the step of the down projections of eight wide experts
        dict(_stack("muon", 8, 14336, 4096, 2048), name="muon_wide_experts"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(round(v / step) * step, math.ceil(lo / step) * step), hi // step * step))


def draw(rng):
    while True:
        kind = rng.choice(["linear", "linear", "decode", "train", "ns", "ns", "muon", "muon"])
        step = rng.choice([1, 8, 64, 64])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        if kind in ("linear", "decode", "train"):
            T = _log(rng, 1, 128) if kind == "decode" else _log(rng, 128, 16384)
            hi = 1024 if dtype == "f32" or step == 1 else 14336
            c = _linear(T, _log(rng, 64, hi, step), _log(rng, 64, hi, step), rng.choice(ACTS), dtype,
                        rng.random() < 0.7, rng.random() < 0.5, kind == "train")
            if work(c)["flops"] <= MAX_LINEAR / (30 if dtype == "f32" else 1):
                return c
        else:
            hi = 768 if dtype == "f32" else 7168
            c = _stack(kind, _log(rng, 1, 128), _log(rng, 32, hi, step), _log(rng, 32, hi, step), _log(rng, 32, 4096),
                       dtype)
            if work(c)["flops"] <= MAX_STACK / (30 if dtype == "f32" else 1) and c["E"] * c["M"] * c["N"] <= MAX_ELEMENTS:
                return c


def work(case):
    c = case
    s = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "linear":
        T, K, N = c["T"], c["K"], c["N"]
        bias, res, train = N * c["bias"], T * N * c["residual"], c["train"]
        moved = T * K + K * N + bias + res + T * N
        if train:  # dy read, the gradients written
            moved += T * N + T * K + K * N + bias
        return {"bytes": s * moved, "flops": 2 * T * K * N * (3 if train else 1)}
    E, S, L = c["E"], min(c["M"], c["N"]), max(c["M"], c["N"])
    # five steps as three and two: a Gram product, symmetric S x S products (half each), one product with X
    flops = E * (6 * S * S * L + 14 * S ** 3)
    if c["kind"] == "ns":
        return {"bytes": 2 * s * E * S * L, "flops": flops}
    return {"bytes": (3 * s + 8) * E * S * L, "flops": flops}


def _gradient(g, E, M, N, rank):
    """Sums of ``rank`` tokens' outer products, their sizes unequal; one matrix of a stack has no tokens."""
    x = torch.randn((E, M, rank), device=DEV, generator=g)
    size = torch.exp(1.5 * torch.randn((E, 1, rank), device=DEV, generator=g)) / rank
    d = torch.empty((E, M, N), device=DEV)
    dy = torch.randn((E, rank, N), device=DEV, generator=g)
    torch.matmul(x * size, dy, out=d)
    if E >= 4:
        d[E // 2].zero_()
    return d


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = DTYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device=DEV, generator=g) * std).to(t)

    s = {"case": c}
    if c["kind"] == "linear":
        T, K, N = c["T"], c["K"], c["N"]
        s["x"], s["w"] = normal(T, K), normal(K, N, std=K ** -0.5)
        s["bias"] = normal(N, std=0.5) if c["bias"] else None
        s["residual"] = normal(T, N) if c["residual"] else None
        if c["train"]:
            s["dy"] = normal(T, N)
            s["leaves"] = [v.requires_grad_(True) for v in (s["x"], s["w"], s["bias"], s["residual"]) if v is not None]
        return s
    E, M, N = c["E"], c["M"], c["N"]
    s["grad"] = _gradient(g, E, M, N, c["rank"]).to(t)
    if c["kind"] == "muon":
        s["param"] = normal(E, M, N, std=0.02)
        s["momentum"] = _gradient(g, E, M, N, c["rank"])
    return s


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    th = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * k * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    c = s["case"]
    t = s["x"].dtype
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        z = x @ w
        if c["bias"]:
            z = z + s["bias"].float()
        y = _act(z, c["act"])
        if c["residual"]:
            y = y + s["residual"].float()
        out = [y.to(t)]
        if c["train"]:
            dy = s["dy"].float()
            dz = dy if c["act"] == "none" else dy * _act_slope(z, c["act"])
            out += [(dz @ w.t()).to(t), (x.t() @ dz).to(t)]
            if c["bias"]:
                out.append(dz.sum(0).to(t))
            if c["residual"]:
                out.append(s["dy"])
        return out


def _plain_ns(x):
    """x: 32 or 64 bits."""
    n = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / (n + EPS).to(x.dtype)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    for _ in range(STEPS):
        a = x @ x.mT
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.mT if tall else x


def _muon_scale(c):
    return math.sqrt(max(1.0, c["N"] / c["M"]))


def run(state):
    s = state
    c = s["case"]
    if c["kind"] == "linear":
        if not own:
            return _plain_linear(s)
        from mintext_amd.kernels import linear
        act = None if c["act"] == "none" else c["act"]
        y = linear(s["x"], s["w"], s["bias"], activation=act, residual=s["residual"])
        return [y] + (list(torch.autograd.grad(y, s["leaves"], s["dy"])) if c["train"] else [])
    # 32 bits lose what a result in 32 bits is held to over five steps: such stacks are computed in 64
    wide = torch.float64 if c["dtype"] == "f32" else torch.float32
    if c["kind"] == "ns":
        if own:
            from mintext_amd.kernels import newton_schulz
            return newton_schulz(s["grad"])
        return _plain_ns(s["grad"].to(wide)).to(s["grad"].dtype)
    if own:
        from mintext_amd.kernels import muon_update
        muon_update(s["param"], s["grad"], s["momentum"], lr=LR, beta=BETA, weight_decay=DECAY)
        return s["param"], s["momentum"]
    g, m = s["grad"].float(), s["momentum"]
    m.mul_(BETA).add_(g, alpha=1 - BETA)
    o = _plain_ns((g * (1 - BETA) + m * BETA).to(wide))
    s["param"].copy_(s["param"].to(wide) * (1 - LR * DECAY) - (LR * _muon_scale(c)) * o)
    return s["param"], m


def _exact_ns(u):
    """One matrix in 64 bits, by the polynomial on its own side."""
    u = u.double()
    u = u / (torch.linalg.vector_norm(u) + EPS)
    for _ in range(STEPS):
        if u.shape[0] <= u.shape[1]:
            g = torch.mm(u, u.t())
            u = torch.mm(torch.addmm(g, g, g, beta=B, alpha=C), u).add_(u, alpha=A)
        else:
            g = torch.mm(u.t(), u)
            u = torch.mm(u, torch.addmm(g, g, g, beta=B, alpha=C)).add_(u, alpha=A)
    return u


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "linear":
        leaves = {k: s[k].detach().double().requires_grad_(c["train"]) for k in ("x", "w", "bias", "residual")
                  if s[k] is not None}
        z = torch.mm(leaves["x"], leaves["w"])
        if c["bias"]:
            z = z + leaves["bias"]
        f = torch.nn.functional
        y = {"none": lambda v: v, "relu": torch.relu, "silu": f.silu, "gelu": f.gelu,
             "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[c["act"]](z)
        if c["residual"]:
            y = y + leaves["residual"]
        out = [y.detach()]
        if c["train"]:
            out += torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
        return out
    if c["kind"] == "ns":
        return torch.stack([_exact_ns(u) for u in s["grad"]])
    g, m = s["grad"].double(), s["momentum"].double()
    m = BETA * m + (1 - BETA) * g
    p = s["param"].double()
    scale = (c["N"] / c["M"]) ** 0.5 if c["N"] > c["M"] else 1.0
    for e in range(c["E"]):
        u = (1 - BETA) * g[e] + BETA * m[e]
        p[e] -= LR * DECAY * p[e] + LR * scale * _exact_ns(u)
    return p, m
