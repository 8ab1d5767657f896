"""Timed cases of the catalogue softmax loss and of the counter-based dropout.

`run` computes each operator either from elementary torch operations (own = False) or with the
package's kernels (own = True), on the same prepared inputs; `exact` gives the same outputs from the
definitions in float64.

  catalogue softmax   x [N, D], w [V, D], labels y [N], scale c, optional row weights a [N]:
      s = c x w^T,  row_n = log sum_v exp(s_nv) - s_n,y_n  (0 where y_n = IGNORE),
      loss = sum_n a_n row_n / Z  with Z = 1 ("sum") or the sum of a over the labelled rows ("mean"),
      and the gradients of the loss by x and w.
  dropout   Philox4x32-10 words of (seed, step, element): y = x / (1 - rate) where the element's word
      is at least round(rate 2^32), else 0, and the same of the upstream gradient.
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100
_PIECE = 1 << 27          # logits per vocabulary piece of the elementary form
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _softmax_case(name, dtype, n, v, d, train=True, scale=1.0, ignored=0.0, weights=False, reduction="sum"):
    return {"name": name, "op": "catalog_softmax", "dtype": dtype, "n": n, "v": v, "d": d, "train": train,
            "scale": scale, "ignored": ignored, "weights": weights, "reduction": reduction}


def _dropout_case(name, dtype, rows, cols, rate):
    return {"name": name, "op": "dropout", "dtype": dtype, "rows": rows, "cols": cols, "rate": rate}


def listed():
    return [
        # one request's log-likelihood under the whole million-item catalogue (no gradient)
        _softmax_case("score_one_f32", "f32", 1, 1_000_000, 128, train=False),
        # the default training batch against the MovieLens-1M catalogue (3706 items + the OOV row)
        _softmax_case("batch_ml1m_f32", "f32", 2048, 3707, 128),
        # unit-norm 64-wide tower outputs at temperature 0.07
        _softmax_case("narrow_f32", "f32", 4096, 20_000, 64, scale=1 / 0.07, reduction="mean"),
        # a large batch against a mid-size catalogue
        _softmax_case("batch_f32", "f32", 8192, 100_000, 128, reduction="mean"),
        # 256-wide towers, sizes that fill no tile
        _softmax_case("wide_f32", "f32", 2999, 30_011, 256),
        # fine-tuning on a handful of rows: the catalogue's bytes bound it
        _softmax_case("few_rows_bf16", "bf16", 64, 200_000, 128, reduction="mean"),
        # a padded batch with sample weights, an odd width
        _softmax_case("ragged_bf16", "bf16", 1021, 50_021, 96, ignored=0.15, weights=True, reduction="mean"),
        # the million-item catalogue in bf16, the largest step
        _softmax_case("catalogue_bf16", "bf16", 16_384, 1_000_000, 128, reduction="mean"),
        # one narrow layer's activations: a launch's latency
        _dropout_case("dropout_small_f32", "f32", 4096, 64, 0.2),
        # a row count and width that fill no vector
        _dropout_case("dropout_odd_f32", "f32", 3701, 333, 0.5),
        # a tower layer at the 65,536-row batch
        _dropout_case("dropout_tower_f32", "f32", 65_536, 256, 0.2),
        # the DCN-v2 ranker's 3344-wide input
        _dropout_case("dropout_wide_bf16", "bf16", 16_384, 3344, 0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    if rng.random() < 0.3:
        rows, cols = _log_int(rng, 1, 65_536), _log_int(rng, 1, 4096)
        rows = max(1, min(rows, 50_000_000 // cols))
        case = _dropout_case("", dtype, rows, cols, rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, 0.9]))
    else:
        d = rng.choice([8, 16, 32, 64, 96, 100, 128, 192, 255, 256, rng.randint(1, 256)])
        v = _log_int(rng, 2, 1_000_000)
        n = _log_int(rng, 1, 16_384)
        cap = 16_384 * 1_000_000 * 128 // 2
        n = max(1, min(n, cap // (v * d)))
        case = _softmax_case("", dtype, n, v, d, train=rng.random() < 0.75,
                             scale=rng.choice([1.0, 0.5, 1 / 0.07, 1 / math.sqrt(d)]),
                             ignored=rng.choice([0.0, 0.0, 0.1, 0.6]), weights=rng.random() < 0.4,
                             reduction=rng.choice(["sum", "mean"]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _softmax_inputs(case, seed):
    """Tower outputs of a partly trained model: a row leans towards its label's item, labels follow
    a popularity law, logits have a standard deviation near 1.5 and the label's one lies near 6."""
    n, v, d = case["n"], case["v"], case["d"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    sigma = math.sqrt(1.5 / (case["scale"] * math.sqrt(d)))
    w = torch.randn((v, d), generator=g, device=dev) * sigma
    y = (v * torch.rand((n,), generator=g, device=dev, dtype=torch.float64) ** 3).to(torch.int64).clamp_(0, v - 1)
    x = torch.randn((n, d), generator=g, device=dev) * sigma
    x += w[y] * (6.0 / (1.5 * math.sqrt(d)))
    if case["ignored"] > 0:
        y = torch.where(torch.rand((n,), generator=g, device=dev) < case["ignored"], torch.full_like(y, IGNORE), y)
    a = 0.25 + 1.5 * torch.rand((n,), generator=g, device=dev) if case["weights"] else None
    dt = _DT[case["dtype"]]
    return x.to(dt), w.to(dt), y, a


def _dropout_inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    shape = (case["rows"], case["cols"])
    dt = _DT[case["dtype"]]
    x = torch.randn(shape, generator=g, device=dev).to(dt)
    dy = (torch.randn(shape, generator=g, device=dev) * 1e-2).to(dt)
    ticket = [int(seed) * 0x9E3779B97F4A7C15 % (1 << 63), int(seed) % 1000]   # (seed, step)
    return x, dy, ticket


def prepare(case, seed):
    if case["op"] == "dropout":
        x, dy, ticket = _dropout_inputs(case, seed)
        return {"case": case, "x": x.requires_grad_(own), "dy": dy,
                "ticket": torch.tensor(ticket, dtype=torch.int64, device=x.device)}
    x, w, y, a = _softmax_inputs(case, seed)
    train = own and case["train"]
    return {"case": case, "x": x.requires_grad_(train), "w": w.requires_grad_(train), "y": y, "a": a}


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    return _own_softmax(state) if own else _plain_softmax(state)


def _own_softmax(state):
    from recsys_amd import functional as F
    case = state["case"]
    if not case["train"]:
        loss, row, lse, _ = F.catalog_softmax_fwd(state["x"], state["w"], state["y"], scale=case["scale"],
                                                  weights=state["a"], ignore_index=IGNORE,
                                                  reduction=case["reduction"], want_grad=False)
        return loss, row, lse
    loss, row = F.catalog_softmax_loss(state["x"], state["w"], state["y"], scale=case["scale"], weights=state["a"],
                                       ignore_index=IGNORE, reduction=case["reduction"])
    dx, dw = torch.autograd.grad(loss, (state["x"], state["w"]))
    return loss.detach(), row, dx, dw


def _own_dropout(state):
    from recsys_amd import functional as F
    y = F.dropout(state["x"], state["case"]["rate"], state["ticket"])
    dx, = torch.autograd.grad(y, (state["x"],), state["dy"])
    return y.detach(), dx


def _plain_softmax(state):
    case = state["case"]
    c = case["scale"]
    x, w = state["x"].float(), state["w"].float()
    n, v = x.shape[0], w.shape[0]
    y = state["y"]
    live = y != IGNORE
    yc = torch.where(live, y, torch.zeros_like(y))
    piece = max(1, min(v, _PIECE // n))
    # the label's own term stays out of the running sum: a small loss is log1p of the others' share
    # and 1 - p of the label their sigmoid, neither a difference of nearly equal numbers
    m = torch.full((n,), -math.inf, device=x.device)
    z = torch.zeros((n,), device=x.device)
    for v0 in range(0, v, piece):
        s = c * (x @ w[v0:v0 + piece].t())
        rows = torch.nonzero(live & (yc >= v0) & (yc < v0 + s.shape[1])).squeeze(1)
        s[rows, yc[rows] - v0] = -math.inf
        m2 = torch.maximum(m, s.amax(1))
        at = torch.where(m2 == -math.inf, torch.zeros_like(m2), m2)
        z = z * torch.exp(m - at) + torch.exp(s - at[:, None]).sum(1)
        m = m2
    others = m + torch.log(z)
    sy = (c * (x.double() * w[yc].double()).sum(1)).float()
    zero = torch.zeros_like(others)
    t = others - sy
    row = torch.where(live, torch.log1p(torch.exp(-t.abs())) + t.clamp(min=0), zero)
    lse = torch.where(live, torch.maximum(others, sy) + torch.log1p(torch.exp(-t.abs())), others)
    short = torch.where(t > 0, 1 / (1 + torch.exp(-t.abs())), torch.exp(-t.abs()) / (1 + torch.exp(-t.abs())))
    a = torch.where(live, state["a"] if state["a"] is not None else torch.ones_like(lse), zero)
    total = (a.double() * row.double()).sum()
    den = a.double().sum() if case["reduction"] == "mean" else torch.ones((), dtype=torch.float64, device=x.device)
    inv = torch.where(den != 0, 1 / den, torch.zeros_like(den))
    loss = (total * inv).float()
    if not case["train"]:
        return loss, row, lse
    r = (a * inv.float()) * c
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for v0 in range(0, v, piece):
        wp = w[v0:v0 + piece]
        p = torch.exp(c * (x @ wp.t()) - lse[:, None])
        rows = torch.nonzero(live & (yc >= v0) & (yc < v0 + wp.shape[0])).squeeze(1)
        p[rows, yc[rows] - v0] = -short[rows]
        p *= r[:, None]
        dx += p @ wp
        dw[v0:v0 + piece] = p.t() @ x
    return loss, row, dx.to(state["x"].dtype), dw.to(state["w"].dtype)


_M0, _M1, _K0, _K1, _U32 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _mul32(m, x):
    """The high and low words of the 64-bit products of m and x (words held in int64)."""
    p0, p1 = m * (x & 0xFFFF), m * (x >> 16)
    return (p1 + (p0 >> 16)) >> 16, (p0 + ((p1 & 0xFFFF) << 16)) & _U32


def _plain_words(n, ticket):
    i = torch.arange((n + 3) // 4, device=ticket.device)
    seed, step = ticket[0], ticket[1]
    k0, k1 = seed & _U32, (seed >> 32) & _U32
    c0, c1 = i & _U32, i >> 32
    c2, c3 = (step & _U32).expand_as(i), ((step >> 32) & _U32).expand_as(i)
    for _ in range(10):
        h0, l0 = _mul32(_M0, c0)
        h1, l1 = _mul32(_M1, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + _K0) & _U32, (k1 + _K1) & _U32
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _plain_dropout(state):
    x, rate = state["x"], state["case"]["rate"]
    keep = (_plain_words(x.numel(), state["ticket"]) >= round(rate * 2.0 ** 32)).reshape(x.shape)
    f = 1.0 / (1.0 - rate)
    zero = torch.zeros((), device=x.device)
    return (torch.where(keep, x.float() * f, zero).to(x.dtype),
            torch.where(keep, state["dy"].float() * f, zero).to(x.dtype))


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the outputs in float64
# ---------------------------------------------------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * es, "flops": 2 * n}
    n, v, d = case["n"], case["v"], case["d"]
    once = (n + v) * d * es + n * 8 + (4 * n if case["weights"] else 0)
    if not case["train"]:
        return {"bytes": once + 8 * n + 4, "flops": 2 * n * v * d}
    return {"bytes": once + (n + v) * d * es + 4 * n + 4, "flops": 6 * n * v * d}


def exact(case, seed):
    if case["op"] == "dropout":
        return _exact_dropout(case, seed)
    x, w, y, a = _softmax_inputs(case, seed)
    x, w = x.double(), w.double()
    n, v, d = case["n"], case["v"], case["d"]
    c = case["scale"]
    labelled = torch.nonzero(y != IGNORE).squeeze(1)
    cols = max(1, min(v, (1 << 26) // n))
    parts = []
    for lo in range(0, v, cols):
        parts.append(torch.logsumexp((x * c) @ w[lo:lo + cols].T, dim=1))
    lse = torch.logsumexp(torch.stack(parts, 1), dim=1)
    row = torch.zeros(n, dtype=torch.float64, device=x.device)
    yl = y[labelled]
    row[labelled] = lse[labelled] - c * torch.einsum("nd,nd->n", x[labelled], w[yl])
    wt = torch.zeros_like(row)
    wt[labelled] = a.double()[labelled] if a is not None else 1.0
    den = float(wt.sum()) if case["reduction"] == "mean" else 1.0
    loss = (wt * row).sum() / den if den else torch.zeros((), dtype=torch.float64, device=x.device)
    if not case["train"]:
        return loss, row, lse
    coef = wt * (c / den if den else 0.0)
    cx = x * coef[:, None]
    dx = torch.zeros_like(x)
    dw = torch.zeros_like(w)
    for lo in range(0, v, cols):
        block = w[lo:lo + cols]
        prob = torch.exp((x * c) @ block.T - lse[:, None])
        dx += prob @ block
        dw[lo:lo + cols] = prob.T @ cx
    dx *= coef[:, None]
    dx[labelled] -= coef[labelled, None] * w[yl]
    dw.index_add_(0, yl, cx[labelled], alpha=-1.0)
    return loss, row, dx, dw


def _exact_dropout(case, seed):
    x, dy, (key, step) = _dropout_inputs(case, seed)
    n = x.numel()
    u32 = np.uint64(_U32)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    ctr = [block & u32, block >> np.uint64(32), np.full_like(block, step & _U32), np.full_like(block, step >> 32)]
    k = [key & _U32, key >> 32]
    for r in range(10):
        a, b = ctr[0] * np.uint64(_M0), ctr[2] * np.uint64(_M1)
        key0 = np.uint64((k[0] + r * _K0) & _U32)
        key1 = np.uint64((k[1] + r * _K1) & _U32)
        ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ key0, b & u32, (a >> np.uint64(32)) ^ ctr[3] ^ key1, a & u32]
    words = np.stack(ctr, axis=1).reshape(-1)[:n]
    keep = torch.from_numpy(words >= np.uint64(round(case["rate"] * 2.0 ** 32))).to(x.device).reshape(x.shape)
    return x.double() * keep / (1.0 - case["rate"]), dy.double() * keep / (1.0 - case["rate"])
