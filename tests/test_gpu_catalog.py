"""Softmax cross entropy over a whole catalogue (csrc/catalog.hip) against the formula in float64.

Tolerances, per element, from the roundings the kernels make:
  logit   |ds| <= c sum_d |x_d w_d| (2^-20 + D 2^-23): the two-term fp16 split drops l l and the third
          term (fp32 inputs; bf16 products are exact), D accumulations of at most one step each
  p       relative 2 |ds| + 2^-20 (exp2, the split of p) + |lse| 2^-22 (the row's lse in fp32 log2 units)
  dX, dW  sum of |terms| times (p's relative error + a step per accumulation), terms p |w| and |w_y|;
          bf16: half a step (2^-8) for each p and for the result
"""
import math

import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
IGN = -100
DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def reference(x, w, y, scale=1.0, weights=None, reduction="sum", g=1.0):
    """float64 loss, row, lse, dX, dW on the CPU, and the sums of magnitudes the tolerances use."""
    x, w, y = x.detach().double().cpu(), w.detach().double().cpu(), y.cpu()
    N = x.shape[0]
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
    return {"loss": (a * row).sum() * inv, "loss_abs": (a.abs() * row.abs()).sum() * inv.abs(),
            "a_abs": a.abs().sum() * inv.abs(), "row": row, "lse": lse, "mag": mag,
            "dx": k * ((p - onehot) @ w), "dw": (k * (p - onehot)).T @ x,
            "dx_abs": k.abs() * (p @ w.abs() + onehot @ w.abs()), "dw_abs": (k.abs() * (p + onehot)).T @ x.abs()}


def tolerances(r, N, V, D, dtype):
    ds = r["mag"] * ((2.0 ** -20 if dtype == torch.float32 else 0.0) + D * 2.0 ** -23)
    rp = 2 * ds + 2.0 ** -20 + r["lse"].abs() * 2.0 ** -22
    rnd = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    acc_x, acc_w = (V / 64 + 64) * 2.0 ** -23, (N / 64 + 64) * 2.0 ** -23
    pr = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    row = 2 * ds + (r["lse"].abs() + 1) * 2.0 ** -21
    rmax = rp.max() if N else torch.tensor(0.0)
    return {"row": row, "loss": float(r["a_abs"]) * (float(row.max()) if N else 0.0) + float(r["loss_abs"]) * 2.0 ** -22,
            "dx": r["dx_abs"] * (rp[:, None] + acc_x + pr) + r["dx"].abs() * rnd + 1e-30,
            "dw": r["dw_abs"] * (rmax + acc_w + pr) + r["dw"].abs() * rnd + 1e-30}


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol).max()), got[bad][:4], want[bad][:4])


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


def step(x, w, y, a=None, scale=1.0, reduction="sum", g=1.0):
    F = pkg("functional")
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, row = F.catalog_softmax_loss(x, w, y, scale, a, IGN, reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(g, device="cuda"))
    return loss.detach(), row, dx, dw


def check(x, w, y, a=None, scale=1.0, reduction="sum", g=1.0):
    F = pkg("functional")
    N, D, V = x.shape[0], x.shape[1], w.shape[0]
    loss, row, dx, dw = step(x, w, y, a, scale, reduction, g)
    l2, row2, lse, _ = F.catalog_softmax_fwd(x, w, y, scale, a, IGN, reduction, want_grad=False)
    r = reference(x, w, y, scale, a, reduction, g)
    t = tolerances(r, N, V, D, x.dtype)
    within(row, r["row"], t["row"], "row")
    within(row2, r["row"], t["row"], "row (loss alone)")
    within(lse, r["lse"], t["row"], "lse")
    within(loss, r["loss"], t["loss"] + 1e-30, "loss")
    within(l2, r["loss"], t["loss"] + 1e-30, "loss alone")
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    within(dx, r["dx"], t["dx"], "dx")
    within(dw, r["dw"], t["dw"], "dw")


@DTYPES
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 2, 8), (2, 1, 64), (1, 5000, 128), (31, 63, 64), (33, 65, 65),
                                   (64, 64, 128), (130, 129, 100), (257, 1000, 256), (700, 333, 129), (65, 20000, 32),
                                   (1500, 70, 96), (513, 4097, 128), (260, 900, 72), (129, 257, 136)])
def test_against_float64(cuda, dtype, N, V, D):
    check(*inputs(N, V, D, dtype, seed=N + V + D)[:3])


@DTYPES
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("N,V,D,scale", [(300, 500, 64, 1 / 0.07), (97, 2500, 128, 0.25), (260, 300, 200, 1.0),
                                         (2048, 60, 64, 0.5), (2049, 300, 128, 0.5), (9000, 40, 64, 1.0)])
def test_weights_ignored_scale(cuda, dtype, reduction, N, V, D, scale):
    x, w, y, a = inputs(N, V, D, dtype, seed=7, ignored=0.4, weights=True, scale=scale)
    check(x, w, y, a, scale, reduction, g=-2.5)


@DTYPES
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
    within(loss, r["loss"], t["loss"], "loss")
    with pytest.raises(ValueError, match="not asked"):
        F.catalog_softmax_bwd(w, state)


@DTYPES
def test_negative_and_zero_weights_and_crowded_labels(cuda, dtype):
    """Half the rows share three labels; weights of both signs and zero."""
    x, w, y, _ = inputs(500, 900, 128, dtype, seed=11)
    y[::2] = torch.tensor([5, 6, 700], device="cuda")[torch.arange(250, device="cuda") % 3]
    a = torch.linspace(-1.0, 1.0, 500, device="cuda")
    a[10:20] = 0.0
    check(x, w, y, a, 1.0, "sum", g=0.5)


@DTYPES
@pytest.mark.parametrize("sx,sw,scale", [(1e18, 1e-18, 1.0), (1e-15, 1e15, 2.0), (1e-20, 1e-12, 1.0), (30.0, 3.0, 1.0)])
def test_magnitudes(cuda, dtype, sx, sw, scale):
    """Far scales of the two operands, logits of zero and of hundreds (a nearly certain item per row)."""
    x, w, y, _ = inputs(90, 400, 96, dtype, seed=5)
    check((x.float() * sx).to(dtype), (w.float() * sw).to(dtype), y, None, scale)


@DTYPES
def test_rows_of_different_scales(cuda, dtype):
    """Each row of x has a scale of its own: small rows keep their relative precision in dX and row loss."""
    x, w, y, _ = inputs(64, 300, 128, dtype, seed=6)
    x = (x.float() * torch.logspace(-6, 1, 64, device="cuda")[:, None]).to(dtype)
    check(x, w, y)


@DTYPES
def test_small_losses_keep_relative_precision(cuda, dtype):
    """A nearly certain label: the loss is about exp(-12), its gradient too; both come relative to
    themselves, not to the logits (bf16: the result's rounding is the whole tolerance left)."""
    F = pkg("functional")
    x, w, y, _ = inputs(40, 200, 64, dtype, seed=8, spread=0.5)
    x = (12.0 * w[y].float() / (w[y].float() ** 2).sum(1, keepdim=True) + 0.1 * x.float()).to(dtype)
    r = reference(x, w, y)
    ds = r["mag"] * (2.0 ** -20 + 64 * 2.0 ** -23)
    loss, row, dx, dw = step(x, w, y)
    assert float(r["row"].max()) < 0.05
    within(row, r["row"], r["row"] * (2 * ds + 2.0 ** -19), "row")
    rnd = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22
    q = 1 - torch.exp(-r["row"])
    # dx = sum over the others of p w - q w_y: both parts carry the factor q
    tol = q[:, None] * (w.double().cpu().abs().amax(0) * 2) * (2 * ds[:, None] + 2.0 ** -18 + rnd) + r["dx"].abs() * rnd
    within(dx, r["dx"], tol, "dx")


@DTYPES
def test_no_rows_all_ignored_and_bad_labels(cuda, dtype):
    x, w, y, _ = inputs(70, 130, 64, dtype, seed=2)
    loss, row, dx, dw = step(x[:0], w, y[:0])
    assert float(loss) == 0 and row.shape == (0,) and dx.shape == (0, 64) and not bool(dw.any())
    for red in ("sum", "mean"):
        loss, row, dx, dw = step(x, w, torch.full_like(y, IGN), reduction=red)
        assert float(loss) == 0 and not bool(row.any()) and not bool(dx.any()) and not bool(dw.any())
    # a label out of range: its row loss, its dX row and the loss are NaN; the other rows are as without it
    for bad in (130, -1, 1 << 40):
        y2 = y.clone()
        y2[13] = bad
        yi = y.clone()
        yi[13] = IGN
        loss, row, dx, dw = step(x, w, y2)
        _, row_i, dx_i, dw_i = step(x, w, yi)
        keep = torch.arange(70, device="cuda") != 13
        assert math.isnan(float(loss)) and math.isnan(float(row[13])) and bool(dx[13].isnan().all())
        assert torch.equal(row[keep], row_i[keep]) and torch.equal(dx[keep], dx_i[keep]) and torch.equal(dw, dw_i)


@DTYPES
def test_ignored_rows_may_hold_anything(cuda, dtype):
    x, w, y, _ = inputs(200, 300, 96, dtype, seed=3, ignored=0.3)
    dead = y == IGN
    x2 = x.clone()
    x2[dead] = float("nan")
    x2[dead, ::3] = float("inf")
    loss, row, dx, dw = step(x, w, y)
    loss2, row2, dx2, dw2 = step(x2, w, y)
    assert torch.equal(loss, loss2) and torch.equal(row, row2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)


@DTYPES
def test_nan_stays_in_its_row(cuda, dtype):
    """A NaN in a labelled row of x: that row's loss and dX, the loss and every item's gradient, no other row."""
    x, w, y, _ = inputs(100, 150, 64, dtype, seed=4)
    x2 = x.clone()
    x2[17, 3] = float("nan")
    _, row, dx, _ = step(x, w, y)
    loss2, row2, dx2, dw2 = step(x2, w, y)
    keep = torch.arange(100, device="cuda") != 17
    assert bool(row2[17].isnan()) and bool(dx2[17].isnan().all()) and bool(loss2.isnan()) and bool(dw2.isnan().all())
    assert torch.equal(row[keep], row2[keep]) and torch.equal(dx[keep], dx2[keep])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradient_against_differences(cuda, D):
    """Central differences of the kernel's own loss along random directions (float32)."""
    F = pkg("functional")
    x, w, y, a = inputs(50, 120, D, torch.float32, seed=9, ignored=0.2, weights=True)
    _, _, dx, dw = step(x, w, y, a, 1.3, "mean")
    g = torch.Generator().manual_seed(1)
    for _ in range(3):
        vx, vw = torch.randn(x.shape, generator=g).cuda(), torch.randn(w.shape, generator=g).cuda()
        h = 2.0 ** -8
        f = [float(F.catalog_softmax_fwd(x + t * h * vx, w + t * h * vw, y, 1.3, a, IGN, "mean", False)[0].double())
             for t in (2, 1, -1, -2)]
        num = (-f[0] + 8 * f[1] - 8 * f[2] + f[3]) / (12 * h)
        ana = float((dx.double() * vx.double()).sum() + (dw.double() * vw.double()).sum())
        # each loss lies between 4 and 8, where a float32 step is 2^-21: four steps each; the formula's own
        # error, h^4 / 30 times a fifth derivative (logits' slopes have a deviation below 10), is below 1e-5
        assert abs(num - ana) <= 18 * 2.0 ** -19 / (12 * h) + 1e-5, (num, ana)


@DTYPES
def test_equal_bits_streams_layouts_and_partial_gradients(cuda, dtype):
    F = pkg("functional")
    x, w, y, a = inputs(300, 1000, 72, dtype, seed=10, weights=True)
    want = step(x, w, y, a, reduction="mean")
    again = step(x, w, y, a, reduction="mean")
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = step(x, w, y, a, reduction="mean")
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    # strided and offset inputs
    xs = torch.zeros((300, 80), dtype=dtype, device="cuda")
    xs[:, 3:75] = x
    wt = w.t().contiguous().t()
    ys = torch.stack([y, y], 1)[:, 0]
    assert all(torch.equal(p, q) for p, q in zip(want, step(xs[:, 3:75], wt, ys, a, reduction="mean")))
    buf = torch.empty(300 * 72 + 1, dtype=dtype, device="cuda")
    xo = buf[1:].view(300, 72).copy_(x)
    assert xo.data_ptr() % 16 != 0
    assert all(torch.equal(p, q) for p, q in zip(want, step(xo, w, y, a, reduction="mean")))
    # one gradient alone, raw calls, a state used twice
    loss, row, lse, state = F.catalog_softmax_fwd(x, w, y, 1.0, a, IGN, "mean", want_grad=(True, False))
    dx, none = F.catalog_softmax_bwd(w, state, dw=False)
    assert none is None and torch.equal(dx, want[2])
    loss, row, lse, state = F.catalog_softmax_fwd(x, w, y, 1.0, a, IGN, "mean", want_grad=(False, True))
    none, dw = F.catalog_softmax_bwd(w, state, dx=False)
    assert none is None and torch.equal(dw, want[3]) and torch.equal(row, want[1])
    _, dw2 = F.catalog_softmax_bwd(w, state, torch.tensor(2.0, device="cuda"), dx=False)
    _, dw3 = F.catalog_softmax_bwd(w, state, dx=False)
    assert torch.equal(dw2.float(), 2 * dw.float()) and torch.equal(dw3, dw)


def test_two_forwards_before_a_backward_and_shared_operands(cuda):
    F = pkg("functional")
    x, w, y, _ = inputs(120, 256, 64, torch.float32, seed=12)
    x1, w1 = x.requires_grad_(True), w.requires_grad_(True)
    l1, _ = F.catalog_softmax_loss(x1, w1, y)
    l2, _ = F.catalog_softmax_loss(x1, w1, (y + 1) % 256, scale=0.5)
    both = torch.autograd.grad(l1 + l2, (x1, w1))
    a1 = step(x, w, y)
    a2 = step(x, w, (y + 1) % 256, scale=0.5)
    for got, p, q in zip(both, a1[2:], a2[2:]):
        assert torch.equal(got, p + q) or torch.equal(got, q + p)
    # rows that are items themselves: one leaf, both gradients
    t = w.detach().clone().requires_grad_(True)
    loss, _ = F.catalog_softmax_loss(t[:120], t, y)
    g, = torch.autograd.grad(loss, (t,))
    ref = step(w.detach()[:120], w, y)
    want = ref[3].clone()
    want[:120] += ref[2]
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError):
        l3, _ = F.catalog_softmax_loss(x1, w1, y)
        gx, = torch.autograd.grad(l3, (x1,), create_graph=True)
        gx.sum().backward()


@DTYPES
def test_captured_and_replayed(cuda, dtype):
    """A captured step, replayed on new contents, against the eager call on the same contents."""
    F = pkg("functional")
    x, w, y, a = inputs(300, 700, 128, dtype, seed=13, weights=True, ignored=0.1)
    bx, bw, by, ba = (t.clone() for t in (x, w, y, a))

    def run():
        loss, row, lse, state = F.catalog_softmax_fwd(bx, bw, by, 2.0, ba, IGN, "mean")
        return (loss, row) + F.catalog_softmax_bwd(bw, state)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for seed in range(3):
        x2, w2, y2, a2 = inputs(300, 700, 128, dtype, seed=20 + seed, weights=True, ignored=0.3)
        for b, t in zip((bx, bw, by, ba), (x2, w2, y2, a2)):
            b.copy_(t)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = step(x2, w2, y2, a2, scale=2.0, reduction="mean")
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(o, want))


@DTYPES
def test_long_catalogue(cuda, dtype):
    """Many splits, the running maximum over 200,000 items; float64 on the device, pieces of the items."""
    N, V, D = 150, 200_003, 64
    x, w, y, _ = inputs(N, V, D, dtype, seed=14, spread=3.0)
    loss, row, dx, dw = step(x, w, y)
    X, W = x.double(), w.double()
    S = X @ W.T
    lse = torch.logsumexp(S, 1)
    P = torch.exp(S - lse[:, None])
    mag = (X.abs() @ W.abs().T).amax(1)
    ds = mag * ((2.0 ** -20 if dtype == torch.float32 else 0.0) + D * 2.0 ** -23)
    rp = 2 * ds + 2.0 ** -20 + lse.abs() * 2.0 ** -22
    rnd = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    pr = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    r = torch.arange(N, device="cuda")
    within(row, (lse - S[r, y]).cpu(), (2 * ds + (lse.abs() + 1) * 2.0 ** -21).cpu(), "row")
    A = P @ W.abs() + W[y].abs()
    G = P @ W - W[y]
    within(dx, G.cpu(), (A * (rp[:, None] + (V / 64 + 64) * 2.0 ** -23 + pr) + G.abs() * rnd).cpu(), "dx")
    A, G = P.T @ X.abs(), P.T @ X
    A.index_add_(0, y, X.abs())
    G.index_add_(0, y, X, alpha=-1.0)
    within(dw, G.cpu(), (A * (rp.max() + 80 * 2.0 ** -23 + pr) + G.abs() * rnd + 1e-30).cpu(), "dw")


def test_offsets_past_32_bits(cuda):
    """A float32 catalogue of more than 2^31 elements (and 2^33 bytes): rows at its far end."""
    if torch.cuda.get_device_properties(0).total_memory < 80 << 30:
        pytest.skip("needs 80 GB")
    N, V, D = 70, 8_500_000, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn((V, D), generator=g, device="cuda").mul_(0.2)
    x = torch.randn((N, D), generator=g, device="cuda").mul_(0.2)
    y = V - 1 - torch.arange(N, device="cuda") * 11
    loss, row, dx, dw = step(x, w, y)
    X = x.double()
    lse = torch.full((N,), -math.inf, dtype=torch.float64, device="cuda")
    for v0 in range(0, V, 500_000):
        lse = torch.logaddexp(lse, torch.logsumexp(X @ w[v0:v0 + 500_000].double().T, 1))
    sy = (X * w[y].double()).sum(1)
    mag = float((X.abs().sum(1) * float(w.abs().max())).max())
    ds = mag * (2.0 ** -20 + D * 2.0 ** -23)
    within(row, (lse - sy).cpu(), 2 * ds + 20 * 2.0 ** -21, "row")
    tail = torch.arange(V - 2000, V, device="cuda")
    P = torch.exp(X @ w[tail].double().T - lse[:, None])
    A, G = P.T @ X.abs(), P.T @ X
    A.index_add_(0, y - (V - 2000), X.abs())
    G.index_add_(0, y - (V - 2000), X, alpha=-1.0)
    within(dw[tail], G.cpu(), (A * (2 * ds + 2.0 ** -19) + G.abs() * 2.0 ** -22 + 1e-30).cpu(), "dw")


def test_refusals(cuda):
    F = pkg("functional")
    x, w, y, a = inputs(8, 16, 64, torch.float32, weights=True)
    with pytest.raises(TypeError):
        F.catalog_softmax_fwd(x.half(), w.half(), y)
    with pytest.raises(TypeError):
        F.catalog_softmax_fwd(x, w.bfloat16(), y)
    with pytest.raises(TypeError):
        F.catalog_softmax_fwd(x, w, y.int())
    with pytest.raises(ValueError, match="contiguous"):
        F.catalog_softmax_fwd(x, w.t().contiguous().t(), y)
    for bad in ((x[:, :32].contiguous(), w, y), (x, w, y[:4]), (x, w[:0], y), (x[0], w, y)):
        with pytest.raises(ValueError):
            F.catalog_softmax_fwd(*bad)
    with pytest.raises(ValueError):
        F.catalog_softmax_fwd(x, w, y, weights=a[:4])
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.catalog_softmax_fwd(x, w, y.cpu())
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e30):
        with pytest.raises(ValueError, match="scale"):
            F.catalog_softmax_fwd(x, w, y, scale=scale)
    with pytest.raises(ValueError, match="reduction"):
        F.catalog_softmax_fwd(x, w, y, reduction="max")
    with pytest.raises(NotImplementedError, match="width"):
        F.catalog_softmax_fwd(torch.zeros((2, 257), device="cuda"), torch.zeros((3, 257), device="cuda"), y[:2])
    with pytest.raises(ValueError, match="weights"):
        F.catalog_softmax_loss(x, w, y, weights=a.clone().requires_grad_(True))
    _, _, _, state = F.catalog_softmax_fwd(x, w, y)
    with pytest.raises(ValueError, match="not the forward's"):
        F.catalog_softmax_bwd(w[:8].contiguous(), state)
    with pytest.raises(ValueError, match="one float32"):
        F.catalog_softmax_bwd(w, state, torch.ones(2, device="cuda"))
