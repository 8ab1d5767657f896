"""The catalogue softmax where rows or items hold values far from the others': rows that take no part,
masked items, items of different scales. Reference and tolerances are test_gpu_catalog's."""
import pytest
import torch

from conftest import pkg
from test_gpu_catalog import DTYPES, IGN, check, inputs, reference, step, tolerances, within

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("N", [200, 2049])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_excluded_rows_may_hold_the_largest_values(cuda, dtype, N, D):
    """Ignored rows, and rows whose label is out of range, reach no item's gradient, whatever finite values
    they hold: their logits pass the type's range."""
    x, w, y, _ = inputs(N, 300, D, dtype, seed=3, ignored=0.3)
    w = (w.float() * 4).to(dtype)
    y[13], y[77] = 300, -1
    dead = (y == IGN) | (y < 0) | (y >= 300)
    clean = torch.where(dead, torch.full_like(y, IGN), y)
    x2 = x.clone()
    g = torch.Generator().manual_seed(1)
    sign = torch.randint(0, 2, x.shape, generator=g).cuda() * 2 - 1
    x2[dead] = (sign * torch.finfo(dtype).max).to(dtype)[dead]
    _, row, dx, dw = step(x, w, clean)
    _, row2, dx2, dw2 = step(x2, w, y)
    assert torch.equal(row[~dead], row2[~dead]) and torch.equal(dx[~dead], dx2[~dead]) and torch.equal(dw, dw2)


def masked(N, V, D, dtype, bias, seed=0):
    """x's last column is 1, w's the item's bias; every seventh item is masked by it. Ignored rows are
    zeros, as a padded batch has them, or favour the masked items. Labels are items that are not masked."""
    x, w, y, _ = inputs(N, V, D, dtype, seed=seed, ignored=0.2)
    x[:, -1] = 1.0
    x[y == IGN, -1] = -1.0
    x[(y == IGN) & (torch.arange(N, device="cuda") % 2 == 0)] = 0.0
    gone = torch.arange(V, device="cuda") % 7 == 3
    w[:, -1] = torch.where(gone, torch.full_like(w[:, -1], bias), 0.25 * w[:, -1])
    y = torch.where(y == IGN, y, torch.where(gone[y.clamp(min=0)], y.clamp(min=0) + 1, y) % V)
    return x, w, y, gone


@DTYPES
@pytest.mark.parametrize("bias", [-1e4, -1e9, -1e30, -3.3e38, -float("inf")])
@pytest.mark.parametrize("N,V,D", [(40, 500, 64), (64, 701, 96), (65, 701, 100), (130, 1000, 128), (300, 259, 256)])
def test_masked_items(cuda, dtype, bias, N, V, D):
    """A masked item changes no other item's logit: loss and gradients are those of the catalogue without it,
    its own gradient is zero. (With an infinite bias the formula has no value in dX's column of the biases.)"""
    F = pkg("functional")
    x, w, y, gone = masked(N, V, D, dtype, bias, seed=N + V)
    at = torch.cumsum(~gone, 0) - 1                      # an item's row among those that are left
    wk, yk = w[~gone], torch.where(y == IGN, y, at[y.clamp(min=0)])
    r = reference(x, wk, yk, 1.0, None, "mean")
    t = tolerances(r, N, V, D, dtype)
    loss, row, dx, dw = step(x, w, y, reduction="mean")
    l2, row2, lse, _ = F.catalog_softmax_fwd(x, w, y, 1.0, None, IGN, "mean", want_grad=False)
    within(row, r["row"], t["row"], "row")
    within(row2, r["row"], t["row"], "row (loss alone)")
    within(loss, r["loss"], t["loss"], "loss")
    within(l2, r["loss"], t["loss"], "loss alone")
    live = (y != IGN).cpu()   # (the others' lse is infinite where they favour a masked item)
    within(lse.cpu()[live], r["lse"][live], t["row"][live], "lse")
    within(dw[~gone], r["dw"], t["dw"], "dw")
    assert not bool(dw[gone].any())
    cols = D - 1 if bias == -float("inf") else D
    within(dx[:, :cols], r["dx"][:, :cols], t["dx"][:, :cols], "dx")


@DTYPES
@pytest.mark.parametrize("N,V,D", [(40, 500, 64), (130, 1000, 128), (300, 600, 256), (70, 5000, 100)])
def test_items_of_different_scales(cuda, dtype, N, V, D):
    """Items from 1e-9 to 1 in size, the larger ones unlikely (a bias of -12): small and large items weigh alike
    in dX, and each item's probability is its own."""
    x, w, y, _ = inputs(N, V, D, dtype, seed=N, spread=1.5)
    x[:, -1] = 1.0
    size = torch.logspace(-9, 0, V, device="cuda")[torch.randperm(V, generator=torch.Generator().manual_seed(2)).cuda()]
    w = (w.float() * size[:, None]).to(dtype)
    w[:, -1] = torch.where(size > 1e-6, torch.full_like(w[:, -1], -12.0), torch.zeros_like(w[:, -1]))
    w[5] = 0.0
    r = reference(x, w, y)
    t = tolerances(r, N, V, D, dtype)
    loss, row, dx, dw = step(x, w, y)
    within(row, r["row"], t["row"], "row")
    within(loss, r["loss"], t["loss"], "loss")
    within(dx, r["dx"], t["dx"], "dx")
    within(dw, r["dw"], t["dw"], "dw")


@pytest.mark.parametrize("sx,sw", [(1e30, 1e-30), (1e-28, 1e28), (1.0, 1e-25)])
def test_far_scales_of_all_items(cuda, sx, sw):
    """The whole catalogue far from one, a zero item in it, with rows that make up for it."""
    x, w, y, _ = inputs(90, 400, 96, torch.float32, seed=5)
    x, w = x * sx, w * sw
    w[7] = 0.0
    r = reference(x, w, y)
    t = tolerances(r, 90, 400, 96, torch.float32)
    loss, row, dx, dw = step(x, w, y)
    within(row, r["row"], t["row"], "row")
    within(dx, r["dx"], t["dx"] + 2.0 ** -126, "dx")
    within(dw, r["dw"], t["dw"] + 2.0 ** -126, "dw")


def test_infinite_and_nan_items(cuda):
    """float32: an item's single infinite entry gives its logit the sign that the row's entry gives it, zero times
    infinity and a NaN entry every row NaN, as the products do; with and without gradients."""
    F = pkg("functional")
    for N in (40, 130):
        x, w, y, _ = inputs(N, 300, 64, torch.float32, seed=N)
        y = torch.where(y == 9, y + 1, y)
        x[:, 3] = x[:, 3].abs() + 0.5
        x[3, 3], x[4, 3] = -0.5, 0.0
        w2 = w.clone()
        w2[9, 3] = -float("inf")
        ref = reference(x, torch.cat([w[:9], w[10:]]), torch.where(y > 9, y - 1, y))
        t = tolerances(ref, N, 300, 64, torch.float32)
        keep = torch.ones(N, dtype=torch.bool)
        keep[3:5] = False
        for row in (step(x, w2, y)[1], F.catalog_softmax_fwd(x, w2, y, want_grad=False)[1]):
            within(row.cpu()[keep], ref["row"][keep], t["row"][keep], "row")
            assert not bool(row[3:5].isfinite().any()) and bool(row[4].isnan())
        w2[9, 3] = float("nan")
        loss, row, dx, dw = step(x, w2, y)
        assert bool(row.isnan().all()) and bool(dx.isnan().all()) and bool(dw.isnan().all())


@DTYPES
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -9, 1.0, 4.0])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (345, 2, 96), (90, 3, 64)])
def test_few_items_of_any_size(cuda, dtype, N, V, D, size):
    """One to three items: no other items' roundings average out those of a probability."""
    x, w, y, _ = inputs(N, V, D, dtype, seed=N, ignored=0.7 if N > 1 else 0.0, scale=0.1)
    check(x, (w.float() * size).to(dtype), y, None, 0.1)
    check(x, (w.float() * size).to(dtype), torch.full_like(y, IGN), None, 0.1)


@DTYPES
@pytest.mark.parametrize("bias", [-1e32, -3.3e38, -float("inf")])
@pytest.mark.parametrize("N", [40, 130])
def test_rows_whose_items_are_all_masked(cuda, dtype, bias, N):
    """Nothing is left to compare the label with: NaN, never a loss of zero; a single item is certain whatever its
    finite logit; a label far above the others, which are masked, is certain too."""
    F = pkg("functional")
    x, w, y, _ = inputs(N, 300, 64, dtype, seed=N)
    x[:, -1] = 1.0
    w[:, -1] = bias
    loss, row, dx, dw = step(x, w, y)
    assert all(bool(t.isnan().all()) for t in (loss, row, dx))
    assert bool(F.catalog_softmax_fwd(x, w, y, want_grad=False)[1].isnan().all())
    if bias > -float("inf"):
        loss, row, dx, dw = step(x, w[:1].contiguous(), torch.zeros_like(y))
        assert not any(bool(t.any()) for t in (loss, row, dx, dw))
    w[7, -1] = 0.0
    loss, row, dx, dw = step(x, w, torch.full_like(y, 7))
    assert not any(bool(t.any()) for t in (loss, row, dx[:, :-1], dw))


@DTYPES
@pytest.mark.parametrize("N,D,scale,size", [(2404, 1, 0.1, 2.0 ** -10), (94, 100, 14.3, 2.0 ** -16), (300, 33, 1.0, 2.0 ** -20)])
def test_an_only_item(cuda, dtype, N, D, scale, size):
    """The log sum of a catalogue of one item is its logit, to the roundings of the terms alone."""
    x, w, y, _ = inputs(N, 1, D, dtype, seed=N, ignored=0.5, scale=scale)
    check(x, (w.float() * size).to(dtype), y, None, scale)


@pytest.mark.parametrize("N,V,D", [(500, 900, 128), (300, 70, 64), (700, 2000, 200)])
@pytest.mark.parametrize("sign", [False, True])
def test_label_terms_of_bf16_items_are_not_rounded(cuda, N, V, D, sign):
    """Labels shared by many rows: an item's gradient is the difference of large label terms -a (1 - p_y) x, which
    keep fp32's precision; half a step (2^-8) is for the result and for the other rows' p alone."""
    x, w, y, _ = inputs(N, V, D, torch.bfloat16, seed=N)
    y = y % 5
    a = torch.linspace(-1.0, 1.5, N, device="cuda") if sign else None
    r = reference(x, w, y, 1.0, a)
    t = tolerances(r, N, V, D, torch.float32)
    _, _, _, dw = step(x, w, y, a)
    X, W, yc = x.double().cpu(), w.double().cpu(), y.cpu()
    P = torch.softmax(X @ W.T, 1)
    P[torch.arange(N), yc] = 0.0
    P *= (a.double().cpu().abs() if sign else torch.ones(N, dtype=torch.float64))[:, None]
    within(dw, r["dw"], t["dw"] + r["dw"].abs() * 2.0 ** -8 + 2.0 ** -8 * (P.T @ X.abs()), "dw")
