"""Softmax cross entropy over a whole catalogue (csrc/catalog.hip) against the formula in float64.

Tolerances, per element, from the roundings the kernels make:
  logit   |ds| <= c sum_d |x_d w_d| (2^-20 + D 2^-23): the two-term fp16 split drops l l and the third
          term (fp32 inputs; bf16 products are exact), D accumulations of at most one step each
  p       relative 2 |ds| + 2^-20 (exp2, the row's lse in fp32 log2 units, the split of p)
  dX, dW  sum of |terms| times (p's relative error + a step per accumulation), terms p |w| and |w_y|;
          bf16: half a step (2^-8) for each p and for the result
"""
import math

import numpy as np
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
IGN = -100


def reference(x, w, y, scale, weights=None, reduction="sum", g=1.0):
    """float64 loss, row, lse, dX, dW and the elementwise tolerances' sums of magnitudes."""
    x, w = x.double().cpu(), w.double().cpu()
    y = y.cpu()
    N, V = x.shape[0], w.shape[0]
    s = scale * x @ w.T
    mag = scale * (x.abs() @ w.abs().T).amax(1) if N else torch.zeros(0, dtype=torch.float64)
    lse = torch.logsumexp(s, 1)
    live = y != IGN
    yc = torch.where(live, y, torch.zeros_like(y))
    a = torch.where(live, weights.double().cpu() if weights is not None else torch.ones(N, dtype=torch.float64),
                    torch.zeros(N, dtype=torch.float64))
    row = torch.where(live, lse - s.gather(1, yc[:, None])[:, 0], torch.zeros_like(lse))
    z = a.sum() if reduction == "mean" else torch.tensor(1.0, dtype=torch.float64)
    inv = 1 / z if z != 0 else torch.zeros_like(z)
    p = torch.exp(s - lse[:, None])
    onehot = torch.zeros_like(p)
    if N:
        onehot[torch.arange(N), yc] = 1.0
    k = (g * scale * inv * a)[:, None]
    return {"loss": (a * row).sum() * inv, "loss_abs": (a.abs() * row.abs()).sum() * inv.abs(), "row": row, "lse": lse,
            "dx": k * ((p - onehot) @ w), "dw": (k * (p - onehot)).T @ x, "mag": mag,
            "dx_abs": k.abs() * (p @ w.abs() + onehot @ w.abs()), "dw_abs": (k.abs() * (p + onehot)).T @ x.abs()}


def tolerances(r, N, V, D, dtype):
    ds = r["mag"] * ((2.0 ** -20 if dtype == torch.float32 else 0.0) + D * 2.0 ** -23)
    rp = 2 * ds + 2.0 ** -20 + r["lse"].abs() * 2.0 ** -22
    rnd = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    acc_x, acc_w = (V / 64 + 64) * 2.0 ** -23, (N / 64 + 64) * 2.0 ** -23
    pr = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    row = 2 * ds + (r["lse"].abs() + 1) * 2.0 ** -21
    rmax = rp.max() if N else torch.tensor(0.0)
    return {"row": row, "dx": r["dx_abs"] * (rp[:, None] + acc_x + pr) + r["dx"].abs() * rnd + 1e-30,
            "dw": r["dw_abs"] * (rmax + acc_w + pr) + r["dw"].abs() * rnd + 1e-30}


def within(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol).max()),
                                 got[bad][:4], want[bad][:4])


def inputs(N, V, D, dtype, seed=0, spread=1.5, ignored=0.0, weights=False, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    sigma = math.sqrt(spread / (scale * math.sqrt(D)))
    x = (torch.randn((N, D), generator=g) * sigma).to(dtype).cuda()
    w = (torch.randn((V, D), generator=g) * sigma).to(dtype).cuda()
    y = torch.randint(0, V, (N,), generator=g)
    if ignored:
        y = torch.where(torch.rand((N,), generator=g) < ignored, torch.full_like(y, IGN), y)
    a = (torch.rand((N,), generator=g) + 0.5).cuda() if weights else None
    return x, w, y.cuda(), a


def check(x, w, y, a=None, scale=1.0, reduction="sum", g=1.0):
    F = pkg("functional")
    N, D, V = x.shape[0], x.shape[1], w.shape[0]
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, row = F.catalog_softmax_loss(x, w, y, scale, a, IGN, reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(g, device="cuda"))
    l2, row2, lse, _ = F.catalog_softmax_fwd(x, w, y, scale, a, IGN, reduction, want_grad=False)
    r = reference(x.detach(), w.detach(), y, scale, a, reduction, g)
    t = tolerances(r, N, V, D, x.dtype)
    within(row, r["row"], t["row"], "row")
    within(row2, r["row"], t["row"], "row (loss alone)")
    within(lse, r["lse"], t["row"], "lse")
    lt = float(r["loss_abs"]) * 2.0 ** -22 + (float(t["row"].max()) * max(1.0, float(r["loss_abs"].abs())) if N else 0)
    lt *= N if reduction == "sum" and N else 1
    assert abs(float(loss) - float(r["loss"])) <= lt + 1e-30
    assert abs(float(l2) - float(r["loss"])) <= lt + 1e-30
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    within(dx, r["dx"], t["dx"], "dx")
    within(dw, r["dw"], t["dw"], "dw")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 2, 8), (2, 1, 64), (1, 5000, 128), (31, 63, 64), (33, 65, 65),
                                   (64, 64, 128), (130, 129, 100), (257, 1000, 256), (700, 333, 129), (65, 20000, 32),
                                   (1500, 70, 96), (513, 4097, 128)])
def test_against_float64(cuda, dtype, N, V, D):
    check(*inputs(N, V, D, dtype, seed=N + V + D)[:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("N,V,D,scale", [(300, 500, 64, 1 / 0.07), (97, 2500, 128, 0.25), (260, 300, 200, 1.0)])
def test_weights_ignored_scale(cuda, dtype, reduction, N, V, D, scale):
    x, w, y, a = inputs(N, V, D, dtype, seed=7, ignored=0.4, weights=True, scale=scale)
    check(x, w, y, a, scale, reduction, g=-2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 15, 17, 33, 64, 65])
@pytest.mark.parametrize("V,D", [(3, 4), (64, 64), (1000, 68), (4099, 128), (700, 256)])
def test_loss_alone(cuda, dtype, N, V, D):
    F = pkg("functional")
    x, w, y, a = inputs(N, V, D, dtype, seed=N + V, ignored=0.2, weights=True)
    r = reference(x, w, y, 1.0, a, "mean")
    t = tolerances(r, N, V, D, dtype)
    loss, row, lse, state = F.catalog_softmax_fwd(x, w, y, 1.0, a, IGN, "mean", want_grad=False)
    within(row, r["row"], t["row"], "row")
    within(lse, r["lse"], t["row"], "lse")
    assert abs(float(loss) - float(r["loss"])) <= float(t["row"].max()) + 2.0 ** -22 * abs(float(r["loss"]))
    with pytest.raises(ValueError, match="not asked"):
        F.catalog_softmax_bwd(w, state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_negative_and_zero_weights_and_crowded_labels(cuda, dtype):
    """Half the rows share three labels; weights of both signs and zero."""
    x, w, y, _ = inputs(500, 900, 128, dtype, seed=11)
    y[::2] = torch.tensor([5, 6, 700], device="cuda")[torch.arange(250, device="cuda") % 3]
    a = torch.linspace(-1.0, 1.0, 500, device="cuda")
    a[10:20] = 0.0
    check(x, w, y, a, 1.0, "sum", g=0.5)
