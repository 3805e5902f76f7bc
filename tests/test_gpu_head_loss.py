"""The head's losses and their gradients against the formulas in 64 bits.

Tolerances.  u is the half step of the operands' type (``finfo(t).eps / 2``), v that of float32.  A float32 sum of n products
is off by at most n v sum |a b|.  With k = 1 / tau:
  ez   = k (D + 2) v (|x| |W|)                          a logit; its largest of a row is mz
  el   = mz + v (8 k max|z| + 4 |lse| + blocks + 64)      the logarithm of the sum: the logits' errors, the exponents' and the
                                                        hardware exponential's roundings, the sum over blocks and lanes
  L    : tau^2 (sum_k p_k ez_k + el + (K + 16) v (|const| + |lse| + sum p |z| k)) + 2 z_loss |lse| el + 4 v |L|
  ed   = |g| unit (front q (ez + el + 16 v (1 + k |z| + |lse|)) + (K + 16) v share) + 4 v |dz|     dz before it is rounded
  dx   : u |dx| + (ed + u |dz|) |W|^T + (V + 8) v |dz| |W|^T;  dW: alike with T terms
The mean's loss is off by the mean of the rows' errors and 4 v of itself.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V_ = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def operands(dev, T, D, V, dtype, order, seed=0, std=1.5):
    g = torch.Generator(device=dev).manual_seed(seed + 7 * T + 3 * D + V)
    x = torch.randn(T, D, device=dev, generator=g).to(dtype)
    w = (torch.randn(V, D, device=dev, generator=g) * (std * D ** -0.5)).to(dtype)
    return x, (w.t() if order == "vd" else w.t().contiguous()), g


def teacher(dev, T, V, K, g, dtype=F32):
    """Entries in no order, some rows clustered, some short, one without any (where there are enough)."""
    near = torch.randint(0, V, (T, 1), device=dev, generator=g)
    step = torch.randint(1, max(V // K, 1) + 1, (T, 1), device=dev, generator=g)
    idx = (near + torch.randperm(K, device=dev, generator=g) * step) % V
    logits = (torch.randn(T, K, device=dev, generator=g) * 2 + 5).to(dtype)
    drop = torch.rand(T, K, device=dev, generator=g) < 0.3
    drop[:, 0] = False
    idx = torch.where(drop, -1, idx)
    if T > 3:
        idx[T // 2] = -7
    return idx, logits


def rows_of(idx, t, tau, V):
    """The teacher's shares [T, V] in 64 bits, sum p log p, and which rows have any."""
    on = (idx >= 0) & ~torch.isneginf(t)
    live = on.any(1)
    e = torch.where(on, t.double() / tau, -math.inf)
    e = torch.where(live[:, None], e, 0.0)
    p = torch.softmax(e, 1) * on * live[:, None]
    share = torch.zeros(len(idx), V, dtype=torch.float64, device=idx.device)
    share.scatter_add_(1, torch.where(on, idx, 0).long(), p)
    const = torch.where(p > 0, p * torch.log(p.clamp(min=1e-300)), 0.0).sum(1)
    return share, const, live


def reference(x, w, share, const, live, tau, z_loss, g, K, half=None):
    """The rows' losses, dx and dW in 64 bits with their tolerances; g: the gradient of each row's loss, half: dz's half step."""
    T, D = x.shape
    V = w.shape[1]
    X, W = x.detach().double(), w.detach().double()
    u, k = torch.finfo(x.dtype).eps / 2, 1 / tau
    z = torch.mm(X, W) * k
    size = torch.mm(X.abs(), W.abs()) * k
    ez = (D + 2) * V_ * size
    lse = torch.logsumexp(z, 1)
    blocks = V / 64 + 4
    el = ez.amax(1) + V_ * (8 * z.abs().amax(1) + 4 * lse.abs() + blocks + 64)
    picked, zs = (share * z).sum(1), (share * z.abs()).sum(1)
    loss = tau ** 2 * (const + lse - picked) + z_loss * lse ** 2
    tl = tau ** 2 * ((share * ez).sum(1) + el + (K + 16) * V_ * (const.abs() + lse.abs() + zs)) + 2 * z_loss * lse.abs() * el
    loss, tl = torch.where(live, loss, 0.0), torch.where(live, tl + 4 * V_ * loss.abs(), 0.0)
    if g is None:
        return (loss, tl)
    unit = (g.double() * tau * live)[:, None]
    front = (1 + 2 * z_loss * lse)[:, None]
    q = torch.exp(z - lse[:, None])
    dz = unit * (front * q - share)
    ed = unit.abs() * (front * q * (ez + el[:, None] + 16 * V_ * (1 + z.abs() + lse.abs()[:, None])) + (K + 16) * V_ * share)
    ed = ed + 4 * V_ * dz.abs()
    er = ed + (u if half is None else half) * dz.abs()
    dx, dw = torch.mm(dz, W.t()), torch.mm(X.t(), dz)
    tx = u * dx.abs() + torch.mm(er + (V + 8) * V_ * dz.abs(), W.abs().t().contiguous())
    tw = u * dw.abs() + torch.mm(X.abs().t().contiguous(), er + (T + 8) * V_ * dz.abs())
    return (loss, tl), (dx, tx), (dw, tw)


def close(got, want, what):
    want, tol = want
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol + 1e-40)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / (tol + 1e-40)).max()):.2f} x"


def check(dev, call, x, w, share, const, live, tau, z_loss, K, seed=5):
    """The loss in each reduction, with and without a gradient, and the gradients for weighted rows and for the mean."""
    T = x.shape[0]
    g = torch.rand(T, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)) + 0.5
    rows, dx, dw = reference(x, w, share, const, live, tau, z_loss, g, K)
    n = max(int(live.sum()), 1)
    with torch.no_grad():
        plain = call(x, w, reduction="none")
    x.requires_grad_(True), w.requires_grad_(True)
    loss = call(x, w, reduction="none")
    assert loss.dtype == torch.float32 and torch.equal(plain, loss.detach())
    close(loss.detach(), rows, "loss")
    gx, gw = torch.autograd.grad(loss, [x, w], g)
    assert gx.dtype == x.dtype and gw.dtype == w.dtype and gw.stride() == w.stride()
    close(gx, dx, "dx")
    close(gw, dw, "dw")
    mean = call(x, w, reduction="mean")
    close(mean.detach(), (rows[0].sum() / n, rows[1].sum() / n + 4 * V_ * rows[0].sum().abs() / n), "mean")
    _, dx, dw = reference(x, w, share, const, live, tau, z_loss, torch.full((T,), 3.0 / n, device=dev), K)
    gx, gw = torch.autograd.grad(mean * 3, [x, w])
    close(gx, dx, "dx of the mean")
    close(gw, dw, "dw of the mean")
    total = call(x.detach(), w.detach(), reduction="sum")
    close(total, (rows[0].sum(), rows[1].sum() + 4 * V_ * rows[0].sum().abs()), "sum")


def check_ce(dev, T, D, V, dtype, order, z_loss=0.0, wide=True, ignored=True, seed=0):
    from mintext_amd.kernels import linear_cross_entropy

    x, w, g = operands(dev, T, D, V, dtype, order, seed)
    y = torch.randint(0, V, (T,), device=dev, generator=g)
    y[0] = V - 1
    live = torch.ones(T, dtype=torch.bool, device=dev)
    if ignored and T > 2:
        live = torch.rand(T, device=dev, generator=g) < 0.7
        live[0], live[1] = True, False
    share = torch.zeros(T, V, dtype=torch.float64, device=dev).scatter_(1, y[:, None], 1.0)
    t = torch.where(live, y, -100).to(torch.int64 if wide else torch.int32)
    call = lambda a, b, reduction: linear_cross_entropy(a, b, t, z_loss=z_loss, reduction=reduction)
    check(dev, call, x, w, share, torch.zeros(T, dtype=torch.float64, device=dev), live, 1.0, z_loss, 1)


def check_kd(dev, T, D, V, K, dtype, order, tau=1.0, wide=False, tdtype=F32, seed=0):
    from mintext_amd.kernels import linear_distillation

    x, w, g = operands(dev, T, D, V, dtype, order, seed)
    idx, t = teacher(dev, T, V, K, g, tdtype)
    share, const, live = rows_of(idx, t, tau, V)
    i = idx.to(torch.int64 if wide else torch.int32)
    call = lambda a, b, reduction: linear_distillation(a, b, i, t, temperature=tau, reduction=reduction)
    check(dev, call, x, w, share, const, live, tau, 0.0, K)


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("T,D,V,K", [(1, 72, 1408, 1), (1, 65, 5003, 90), (4, 264, 2056, 1), (20, 1001, 999, 33), (64, 128, 4100, 1),
                                     (50, 130, 3001, 7), (63, 512, 777, 1)])
def test_few_rows_dz_in_two_planes(dev, T, D, V, K, order):
    """dz of few rows is held as its rounding and the rounded rest: what is left is u times at most u |dz|, u = 2^-8."""
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, gen = operands(dev, T, D, V, BF, order, 11)
    g = torch.rand(T, device=dev, generator=gen) + 0.5
    if K == 1:
        y = torch.randint(0, V, (T,), device=dev, generator=gen)
        live = torch.arange(T, device=dev) % 5 != 3
        share = torch.zeros(T, V, dtype=torch.float64, device=dev).scatter_(1, y[:, None], 1.0)
        const, tau = torch.zeros(T, dtype=torch.float64, device=dev), 1.0
        call = lambda a, b: linear_cross_entropy(a, b, torch.where(live, y, -100), z_loss=1e-3, reduction="none")
    else:
        idx, t = teacher(dev, T, V, K, gen, F32)
        tau = 0.5
        share, const, live = rows_of(idx, t, tau, V)
        call = lambda a, b: linear_distillation(a, b, idx, t, temperature=tau, reduction="none")
    _, dx, dw = reference(x, w, share, const, live, tau, 1e-3 if K == 1 else 0.0, g, K, half=2.0 ** -16)
    gx, gw = torch.autograd.grad(call(x.requires_grad_(True), w.requires_grad_(True)), [x, w], g)
    close(gx, dx, "dx")
    close(gw, dw, "dw")


@pytest.mark.parametrize("order", ["dv", "vd"])
def test_gradient_of_logits_far_from_zero(dev, order):
    """f32 logits of 4096 + n / 128 are exact here, and what softmax has to do with is their distance from the largest alone:
    q is off by 16 v (1 + that) and the sum's v (blocks + 64), however large they are."""
    from mintext_amd.kernels import linear_cross_entropy

    T, V = 3, 1000
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.tensor([[64.0, 1.0], [64.0, 0.5], [64.0, -1.0]], device=dev)
    n = torch.randint(-256, 256, (V,), device=dev, generator=g) / 64
    w = torch.stack([torch.full_like(n, 64.0), n])
    w = w.t().contiguous().t() if order == "vd" else w
    y = torch.tensor([1, V - 1, 500], device=dev)
    z = torch.mm(x.double(), w.double())
    far = z.amax(1, keepdim=True) - z
    q = torch.softmax(z, 1)
    dz = q - torch.zeros_like(q).scatter_(1, y[:, None], 1.0)
    ed = q * V_ * (16 * (1 + far) + V / 64 + 64) + 4 * V_ * dz.abs()
    for t in range(T):
        x1, w1 = x[t:t + 1].clone().requires_grad_(True), w.detach().requires_grad_(True)
        gx, gw = torch.autograd.grad(linear_cross_entropy(x1, w1, y[t:t + 1], reduction="sum"), [x1, w1])
        X, W = x1.detach().double(), w1.detach().double()
        close(gw, (torch.mm(X.t(), dz[t:t + 1]), torch.mm(X.abs().t(), ed[t:t + 1] + 4 * V_ * dz[t:t + 1].abs())), "dw")
        close(gx, (torch.mm(dz[t:t + 1], W.t()),
                   torch.mm(ed[t:t + 1] + (V + 8) * V_ * dz[t:t + 1].abs(), W.abs().t().contiguous())), "dx")


# few rows; small tiles that hang over; large tiles (more than 192 of them) with whole and cut stages; odd widths and vocabularies
SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 40, 264), (17, 64, 1000), (61, 136, 4099), (64, 256, 512), (65, 264, 777),
         (129, 512, 2056), (300, 520, 5003), (257, 72, 20011), (1000, 1001, 999), (513, 2048, 1537)]
LARGE = [(4099, 72, 4104), (4099, 65, 4103), (2048, 128, 6400), (3001, 264, 5120)]


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_cross_entropy(dev, size, dtype, order):
    n = SIZES.index(size)
    check_ce(dev, *size, dtype, order, 1e-3 if n % 2 else 0.0, n % 3 == 0)


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("size", LARGE)
def test_cross_entropy_large_tiles(dev, size, order):
    check_ce(dev, *size, BF, order, 1e-3)


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", [(1, 8, 8, 1), (5, 40, 264, 3), (61, 136, 4099, 64), (70, 264, 777, 100), (300, 520, 5003, 17),
                                  (33, 64, 2000, 1024), (257, 72, 20011, 50)])
def test_distillation(dev, size, dtype, order):
    n = size[0] % 3
    check_kd(dev, *size, dtype, order, (1.0, 2.0, 0.5)[n], n == 1, BF if n == 2 else F32)


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("size", [(4099, 72, 4104, 20), (4099, 65, 4103, 64), (3001, 264, 5120, 7)])
def test_distillation_large_tiles(dev, size, order):
    check_kd(dev, *size, BF, order, 2.0)


@pytest.mark.parametrize("order", ["dv", "vd"])
@pytest.mark.parametrize("size", [(16384, 64, 40000), (16411, 40, 39001)])
def test_pieces_of_the_vocabulary(dev, size, order):
    """More than 1 GiB of logits: dx is summed over two pieces, in two shares of each."""
    from mintext_amd import _lib as L

    T, D, V = size
    assert L.query("mtx_head_loss_workspace_size", L.MTX_BF16, T, D, V, int(order == "vd"), 1) < 2 * T * V
    check_ce(dev, T, D, V, BF, order)


def test_pieces_in_32_bits(dev):
    check_kd(dev, 16390, 24, 20000, 5, F32, "dv")


@pytest.mark.parametrize("order", ["dv", "vd"])
def test_weight_beyond_32_bits_of_offset(dev, order):
    """2.2e9 weights: the last columns' logits and gradients."""
    from mintext_amd.kernels import linear_cross_entropy

    T, D, V, n = 5, 2104, 1050000, 1000
    x = torch.randn(T, D, device=dev).to(BF)
    table = torch.zeros((V, D) if order == "vd" else (D, V), device=dev, dtype=BF)
    w = table.t() if order == "vd" else table
    w[:, V - n:] = (torch.randn(D, n, device=dev) * D ** -0.5).to(BF)
    y = torch.tensor([V - 1, V - n, V - 7, 0, V - 100], device=dev)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, y, reduction="none")
    gx, gw = torch.autograd.grad(loss.sum(), [x, w])
    # the columns before the last n all have logit 0
    X, W = x.detach().double(), w.detach()[:, V - n:].double()
    z = X @ W
    lse = torch.log(torch.exp(z).sum(1) + (V - n))
    pick = torch.where(y >= V - n, z.gather(1, (y - (V - n)).clamp(min=0)[:, None])[:, 0], 0.0)
    # the logits' errors (D + 2) v |x| |w| are below 3e-3 here; the sum of 16400 blocks another 16500 v
    tol = (D + 2) * V_ * (X.abs() @ W.abs()).amax() + 16500 * V_
    assert (loss.detach().double() - (lse - pick)).abs().max() <= 2 * tol
    dz = torch.exp(z - lse[:, None])
    dz[y >= V - n] -= torch.nn.functional.one_hot((y - (V - n)).clamp(min=0), n)[y >= V - n].double()
    dx, dw = dz @ W.t(), X.t() @ dz
    er = dz.abs() * 2.0 ** -8 + 2 * tol * torch.exp(z - lse[:, None])
    assert ((gx.double() - dx).abs() <= 2.0 ** -8 * dx.abs() + er @ W.abs().t() + n * V_ * (dz.abs() @ W.abs().t())).all()
    assert ((gw[:, V - n:].double() - dw).abs() <= 2.0 ** -8 * dw.abs() + X.abs().t() @ er + 8 * V_ * (X.abs().t() @ dz.abs())).all()
    # before them every column's gradient is the same, 1 / sum, but for column 0's own target
    first = (X.t() @ (torch.exp(-lse)[:, None] * torch.ones(T, 1, device=dev).double()))
    part = gw[:, 5:V - n:(V - n) // 300].double()
    assert ((part - first).abs() <= 2.0 ** -8 * first.abs() + (2.0 ** -8 + 2 * tol) * (X.abs().t() @ torch.exp(-lse)[:, None])).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_a_class(dev, dtype):
    """All ignored; one that is out of range; a teacher's empty rows, -inf, the type's lowest value, and NaN in empty places."""
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, g = operands(dev, 6, 40, 300, dtype, "dv")
    x.requires_grad_(True), w.requires_grad_(True)
    none = torch.full((6,), -100, device=dev)
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, none, reduction=reduction)
        gx, gw = torch.autograd.grad(loss.sum(), [x, w])
        assert not loss.any() and not gx.any() and not gw.any()
    # another ignored class, a valid index among them
    y = torch.tensor([3, 0, 3, 299, 3, 3], device=dev)
    a = linear_cross_entropy(x, w, y, ignore_index=3, reduction="none")
    b = linear_cross_entropy(x, w, torch.where(y == 3, -100, y), reduction="none")
    assert torch.equal(a, b) and not a[y == 3].any() and (a[y != 3] > 0).all()
    for wrong in (300, -1, 1 << 40, -(1 << 40)):
        loss = linear_cross_entropy(x, w, torch.tensor([1, wrong, 2, -100, 4, 5], device=dev), reduction="none")
        gx, gw = torch.autograd.grad(loss, [x, w], torch.ones(6, device=dev))
        assert torch.isnan(loss).tolist() == torch.isnan(gx).any(1).tolist() == [False, True, False, False, False, False]
        assert torch.isnan(gw).all() and not gx[3].any()
    # an ignored row's x may be anything as far as the losses and dx go
    odd = x.detach().clone()
    odd[3, 5], odd[1] = float("nan"), float("inf")
    odd.requires_grad_(True)
    t = torch.tensor([1, -100, 2, -100, 4, 5], device=dev)
    loss = linear_cross_entropy(odd, w, t, reduction="none")
    (gx,) = torch.autograd.grad(loss.sum(), [odd])
    want = linear_cross_entropy(x, w, t, reduction="none")
    assert torch.equal(loss, want) and torch.equal(gx, torch.autograd.grad(want.sum(), [x])[0])

    idx = torch.tensor([[5, 9, 0], [-1, -1, -1], [7, -1, 2], [1, 2, 3], [8, 299, 8], [4, 5, 6]], device=dev)
    lowest = torch.finfo(torch.float32).min
    inf, nan = float("inf"), float("nan")
    t = torch.tensor([[1.0, 2, -inf], [nan, inf, 3], [2, nan, 1], [-inf, -inf, -inf], [1, 2, 3], [lowest, lowest, 0.5]], device=dev)
    clean = [([5, 9], [1.0, 2]), None, ([7, 2], [2.0, 1]), None, ([8, 299, 8], [1.0, 2, 3]), ([6], [0.5])]
    loss = linear_distillation(x, w, idx, t, reduction="none")
    gx, gw = torch.autograd.grad(loss.sum(), [x, w])
    assert torch.isfinite(loss).all() and torch.isfinite(gx).all() and torch.isfinite(gw).all()
    for r, entry in enumerate(clean):
        if entry is None:
            assert loss[r] == 0 and not gx[r].any()
            continue
        one = linear_distillation(x[r:r + 1], w, torch.tensor([entry[0]], device=dev), torch.tensor([entry[1]], device=dev),
                                  reduction="none")
        (g1,) = torch.autograd.grad(one.sum(), [x])
        # the same numbers; the shares' sums are taken in another order
        assert torch.allclose(one, loss[r:r + 1], rtol=32 * V_, atol=32 * V_)
        assert (g1[r].double() - gx[r].double()).abs().max() <= 2 * torch.finfo(dtype).eps * gx[r].abs().max()
    mean = linear_distillation(x, w, idx, t)
    assert torch.allclose(mean, loss.sum() / 4, rtol=8 * V_)
    empty = linear_distillation(x, w, torch.full((6, 2), -1, device=dev), torch.zeros(6, 2, device=dev))
    gx, gw = torch.autograd.grad(empty, [x, w])
    assert empty == 0 and not gx.any() and not gw.any()
    bad = linear_distillation(x, w, torch.where(idx == 299, 300, idx), t, reduction="none")
    assert torch.isnan(bad).tolist() == [False, False, False, False, True, False]
    t[0, 1] = nan  # of an entry that counts
    bad = linear_distillation(x, w, idx, t, reduction="none")
    assert torch.isnan(bad).tolist() == [True, False, False, False, False, False]


@pytest.mark.parametrize("tau", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("tdtype", [F32, BF])
def test_teacher_logits_of_the_lowest_value(dev, tau, tdtype):
    """They are left out beside others, as their share is 0, and alone are all alike."""
    from mintext_amd.kernels import linear_distillation

    x, w, g = operands(dev, 3, 40, 300, F32, "dv")
    low = torch.finfo(tdtype).min
    idx = torch.tensor([[5, 9, 77, 250], [1, 2, 3, 4], [8, 299, 0, -1]], device=dev)
    t = torch.tensor([[low] * 4, [low, 2.0, low, 1.0], [low] * 4], device=dev).to(tdtype)
    same = torch.tensor([[0.0] * 4, [-float("inf"), 2.0, -float("inf"), 1.0], [0.0] * 4], device=dev)
    a = linear_distillation(x, w, idx, t, temperature=tau, reduction="none")
    assert torch.isfinite(a).all() and torch.equal(a, linear_distillation(x, w, idx, same, temperature=tau, reduction="none"))


def test_backward_twice(dev):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, g = operands(dev, 70, 64, 500, BF, "vd")
    x.requires_grad_(True), w.requires_grad_(True)
    y = torch.randint(0, 500, (70,), device=dev, generator=g)
    idx, t = teacher(dev, 70, 500, 9, g)
    for loss in (linear_cross_entropy(x, w, y), linear_distillation(x, w, idx, t)):
        first = torch.autograd.grad(loss, [x, w], retain_graph=True)
        half = torch.autograd.grad(loss / 2, [x, w], retain_graph=True)
        again = torch.autograd.grad(loss, [x, w])
        assert all(torch.equal(a, b) and torch.equal(a, 2 * c) for a, b, c in zip(first, again, half))


def test_one_entry_is_cross_entropy(dev):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, g = operands(dev, 200, 136, 3001, BF, "vd")
    y = torch.randint(0, 3001, (200,), device=dev, generator=g)
    y[5] = -100
    a = linear_cross_entropy(x, w, y, reduction="none")
    b = linear_distillation(x, w, torch.where(y < 0, -1, y)[:, None], torch.randn(200, 1, device=dev, generator=g), reduction="none")
    assert torch.equal(a, b)
    # twice the same class, each with half of the probability: two terms of p log p, log 2 less, and the same gradient
    x.requires_grad_(True)
    twice = torch.where(y < 0, -1, y)[:, None].expand(200, 2)
    c = linear_distillation(x, w, twice, torch.zeros(200, 2, device=dev), reduction="none")
    off = (a.double() - c.detach().double() - torch.where(y < 0, 0.0, math.log(2))).abs().max()
    assert off <= 16 * V_ * (1 + a.abs().max())
    g1 = torch.autograd.grad(c.sum(), [x])[0]
    g2 = torch.autograd.grad(linear_cross_entropy(x, w, y, reduction="none").sum(), [x])[0]
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("size", [(50, 64, 300), (50, 33, 301)])
def test_infinities_and_nan(dev, size):
    """They reach the rows that they reach in the formula, and no others."""
    from mintext_amd.kernels import linear_cross_entropy

    T, D, V = size
    x, w, g = operands(dev, T, D, V, BF, "dv")
    y = torch.randint(0, V, (T,), device=dev, generator=g)
    clean = linear_cross_entropy(x, w, y, reduction="none")
    x[3, 5], x[T - 1, D - 1] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[3] = keep[T - 1] = False
    assert torch.equal(loss[keep], clean[keep]) and torch.isnan(loss[3]) and not torch.isfinite(loss[T - 1])
    # logits far apart: the sum neither overflows nor vanishes
    big = (x[:3].float() * 1000).to(BF)
    loss = linear_cross_entropy(big, w, y[:3], reduction="none")
    want = torch.nn.functional.cross_entropy(big.double() @ w.double(), y[:3], reduction="none")
    assert ((loss.double() - want).abs() <= (D + 20) * V_ * 2 * (big.double().abs() @ w.double().abs()).amax(1)).all()


def test_shapes_strides_and_alignment(dev):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, g = operands(dev, 24, 64, 320, BF, "dv")
    y = torch.randint(0, 320, (24,), device=dev, generator=g)
    idx, t = teacher(dev, 24, 320, 4, g)
    ce, kd = linear_cross_entropy(x, w, y, reduction="none"), linear_distillation(x, w, idx, t, reduction="none")
    x3 = x.reshape(6, 4, 64).permute(1, 0, 2).contiguous().permute(1, 0, 2)  # [6, 4, 64], not contiguous
    wide = torch.zeros(64, 640, device=dev, dtype=BF)
    wide[:, ::2] = w
    off = torch.empty(1 + 64 * 320, device=dev, dtype=BF)[1:].view(64, 320).copy_(w)
    table = torch.empty(3 + 64 * 320, device=dev, dtype=BF)[3:].view(320, 64).copy_(w.t())
    xo = torch.empty(5 + 24 * 64, device=dev, dtype=BF)[5:].view(6, 4, 64).copy_(x.view(6, 4, 64))
    for a in (x3, xo):
        for b in (w, wide[:, ::2], off, table.t(), w.t().contiguous().t()):
            got = linear_cross_entropy(a, b, y.view(6, 4), reduction="none")
            assert got.shape == (6, 4) and torch.equal(got.reshape(-1), ce)
            got = linear_distillation(a, b, idx.view(6, 4, 4), t.view(6, 4, 4), reduction="none")
            assert torch.equal(got.reshape(-1), kd)
    one = linear_cross_entropy(x[0], w, y[0], reduction="none")
    assert one.shape == () and torch.equal(one, ce[0])
    # gradients in each layout, a gradient that is an expanded scalar, and a weight used twice
    grads = []
    for b in (w, wide[:, ::2], off, table.t()):
        a, b = x.clone().requires_grad_(True), b.detach().requires_grad_(True)
        gx, gw = torch.autograd.grad(linear_cross_entropy(a, b, y, reduction="none").sum(), [a, b])
        grads.append((gx, gw))
    for gx, gw in grads[1:]:
        assert torch.equal(gx, grads[0][0]) and torch.equal(gw, grads[0][1])
    b = w.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(linear_cross_entropy(x, b, y) + linear_cross_entropy(x, b, y), [b])
    (g1,) = torch.autograd.grad(linear_cross_entropy(x, b, y), [b])
    assert torch.equal(gw, 2 * g1)


def test_empty(dev):
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w = torch.empty(0, 40, device=dev, requires_grad=True), torch.randn(40, 70, device=dev, requires_grad=True)
    y = torch.empty(0, dtype=torch.int64, device=dev)
    i, t = torch.empty(0, 3, dtype=torch.int32, device=dev), torch.empty(0, 3, device=dev)
    for f in (lambda r: linear_cross_entropy(x, w, y, reduction=r), lambda r: linear_distillation(x, w, i, t, reduction=r)):
        for r in ("mean", "sum", "none"):
            loss = f(r)
            assert loss.shape == ((0,) if r == "none" else ()) and not loss.any()
            gx, gw = torch.autograd.grad(loss.sum(), [x, w])
            assert gx.shape == (0, 40) and not gw.any()


def test_only_what_is_asked_for(dev):
    from mintext_amd.kernels import linear_cross_entropy

    x, w, g = operands(dev, 70, 64, 500, BF, "dv")
    y = torch.randint(0, 500, (70,), device=dev, generator=g)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    full = torch.autograd.grad(linear_cross_entropy(a, b, y), [a, b])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, y), [a])[0], full[0])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, b, y), [b])[0], full[1])
    # the results may be changed in place before the backward pass
    for reduction in ("mean", "none"):
        loss = linear_cross_entropy(a, b, y, reduction=reduction)
        want = torch.autograd.grad(2 * linear_cross_entropy(a, b, y, reduction=reduction).sum(), [a, b])
        loss *= 2
        assert all(torch.equal(i, j) for i, j in zip(torch.autograd.grad(loss.sum(), [a, b]), want))
    (gx,) = torch.autograd.grad(linear_cross_entropy(a, b, y), [a], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), [a])


@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_gradient_against_differences(dev, kind):
    """The slope along a random direction, of the formula in 64 bits: a step of 1e-5 leaves 1e-10 of third derivatives and 1e-16 /
    1e-5 of rounding, of sums of size below 1e4."""
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    T, D, V, K, step = 12, 24, 90, 4, 1e-5
    x, w, g = operands(dev, T, D, V, F32, "dv")
    if kind == "ce":
        y = torch.randint(0, V, (T,), device=dev, generator=g)
        tau, zl, K = 1.0, 1e-2, 1
        share, const, live = torch.nn.functional.one_hot(y, V).double(), torch.zeros(T, device=dev).double(), y >= 0
        loss = lambda a, b: linear_cross_entropy(a, b, y, z_loss=zl, reduction="sum")
    else:
        idx, t = teacher(dev, T, V, K, g)
        tau, zl = 2.0, 0.0
        share, const, live = rows_of(idx, t, tau, V)
        loss = lambda a, b: linear_distillation(a, b, idx, t, temperature=tau, reduction="sum")
    _, dx, dw = reference(x, w, share, const, live, tau, zl, torch.ones(T, device=dev), K)
    x.requires_grad_(True), w.requires_grad_(True)
    grads = torch.autograd.grad(loss(x, w), [x, w])
    for n, (leaf, (_, tol)) in enumerate(((x, dx), (w, dw))):
        move = torch.randn(*leaf.shape, device=dev, generator=g).double()

        def f(s):
            a, b = (v.detach().double() + (s * step * move if i == n else 0) for i, v in enumerate((x, w)))
            z = (a @ b) / tau
            lse = torch.logsumexp(z, 1)
            return (live * (tau ** 2 * (const + lse - (share * z).sum(1)) + zl * lse ** 2)).sum()

        slope, want = (f(1) - f(-1)) / (2 * step), (grads[n].double() * move).sum()
        assert (slope - want).abs() <= (tol * move.abs()).sum() + 1e-6 * (1 + (grads[n].double() * move).abs().sum())


@pytest.mark.parametrize("size", [(1, 64, 1000), (61, 136, 2003), (700, 256, 4096)])
@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_streams_and_graph(dev, kind, size):
    """Another stream, repeated calls bit for bit, and a captured step replayed between eager ones."""
    from mintext_amd.kernels import linear_cross_entropy, linear_distillation

    x, w, g = operands(dev, *size, BF, "vd")
    y = torch.randint(0, size[2], (size[0],), device=dev, generator=g)
    idx, t = teacher(dev, size[0], size[2], 8, g)
    x2 = torch.flip(x, [1]).contiguous()

    def step(v):
        a, b = v.detach().requires_grad_(True), w.detach().requires_grad_(True)  # leaves of its own: no graph outlives a call
        loss = linear_cross_entropy(a, b, y) if kind == "ce" else linear_distillation(a, b, idx, t, temperature=2.0)
        return [loss.detach()] + list(torch.autograd.grad(loss, [a, b]))

    same = lambda a, c: all(torch.equal(i, j) for i, j in zip(a, c))
    want, want2 = step(x), step(x2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert same(step(x), want)
    torch.cuda.current_stream().wait_stream(side)
    held = x.clone()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    with torch.cuda.graph(graph2, pool=graph.pool()):
        out2 = step(held)
    for v, r in ((x, want), (x2, want2), (x, want), (x2, want2)):
        held.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, r) and same(step(v), r)
        graph2.replay()
        torch.cuda.synchronize()
        assert same(out2, r)


def test_jit_trace_computes(dev):
    from mintext_amd.kernels import linear_cross_entropy

    x, w, g = operands(dev, 20, 64, 300, BF, "dv")
    y = torch.randint(0, 300, (20,), device=dev, generator=g)
    f = lambda a: linear_cross_entropy(a, w, y, reduction="none")
    assert torch.equal(torch.jit.trace(f, (x,), check_trace=False)(-x), f(-x))
