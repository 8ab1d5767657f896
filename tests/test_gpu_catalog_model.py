"""Dropout between a tower's layers and the loss over the encoded catalogue, used together
(models.MultiTowerModel.catalog_loss), against the same computation in float64 on the CPU with the masks
of a numpy Philox."""
import numpy as np
import pytest
import torch

from conftest import pkg
from test_gpu_dropout import kept

pytestmark = pytest.mark.gpu
NU, NI, D = 40, 150, 64


def build(dropout, precision=0, seed=3):
    cfg = pkg("config").ModelConfig(embedding_dim=D, user_tower_dims=[96, 32], item_tower_dims=[96, 32],
                                    contraction_precision=precision)
    m = pkg("models").MultiTowerModel(cfg, [str(i) for i in range(NU)], [str(i) for i in range(NI)], {}, seed=seed,
                                      device="cuda", tower_dropout=dropout)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for t in (m.user_tower, m.item_tower):
            for l in t.layers:
                l.bias.copy_(torch.randn(l.bias.shape, generator=g) * 0.1)
        for e in (m.user_embedding, m.item_embedding):
            e.weight.copy_(torch.randn(e.weight.shape, generator=g) * 0.5)
    return m


def batch(B, seed=0):
    g = torch.Generator().manual_seed(seed)
    return {"user_id": torch.randint(0, NU + 1, (B,), generator=g).cuda(),
            "movie_id": torch.randint(0, NI + 1, (B,), generator=g).cuda()}


def tower64(x, tower, states, P, name):
    h = x
    n = len(tower.layers)
    for j in range(n):
        h = h @ P[f"{name}.{j}.kernel"] + P[f"{name}.{j}.bias"]
        if j < n - 1:
            h = torch.relu(h)
            if states is not None:
                seed, step, rate = states[j]
                h = torch.where(kept(h.shape, rate, seed, step), h / (1 - rate), torch.zeros_like(h))
    return h


def reference(m, feats, states, scale, ignore, reduction):
    P = {}
    for name, t in (("u", m.user_tower), ("i", m.item_tower)):
        for j, l in enumerate(t.layers):
            P[f"{name}.{j}.kernel"] = l.kernel.detach().double().cpu().requires_grad_(True)
            P[f"{name}.{j}.bias"] = l.bias.detach().double().cpu().requires_grad_(True)
    ue = m.user_embedding.weight.detach().double().cpu().requires_grad_(True)
    ie = m.item_embedding.weight.detach().double().cpu().requires_grad_(True)
    uid, iid = feats["user_id"].cpu(), feats["movie_id"].cpu()
    u = tower64(ue[uid], m.user_tower, states and states["u"], P, "u")
    c = tower64(ie, m.item_tower, states and states["i"], P, "i")
    c.retain_grad()
    s = scale * u @ c.T
    row = torch.logsumexp(s, 1) - s.gather(1, iid[:, None])[:, 0]
    live = (iid != ignore).double()
    loss = (row * live).sum() / (live.sum() if reduction == "mean" else 1.0)
    loss.backward()
    return loss.detach(), P, ue.grad, ie.grad, c.grad


@pytest.mark.parametrize("dropout", [0.0, 0.3])
@pytest.mark.parametrize("reduction,ignore", [("mean", 0), ("sum", -100)])
def test_catalog_loss_against_float64(cuda, dropout, reduction, ignore):
    m = build(dropout)
    feats = batch(96)
    states = None
    if dropout:
        states = {"u": [tuple(d.state.tolist()) + (dropout,) for d in m.user_tower.dropouts],
                  "i": [tuple(d.state.tolist()) + (dropout,) for d in m.item_tower.dropouts]}
    loss = m.catalog_loss(feats, scale=0.7, ignore_index=ignore, reduction=reduction)
    loss.backward()
    want, P, gu, gi, gc = reference(m, feats, states, 0.7, ignore, reduction)
    # float32 GEMMs of at most 96 terms over three layers each way, then the loss's own 2^-18: 1e-4 of
    # each tensor's largest entry is ten times their sum
    assert abs(float(loss.detach()) - float(want)) <= 1e-5 * abs(float(want))
    for name, t in (("u", m.user_tower), ("i", m.item_tower)):
        for j, l in enumerate(t.layers):
            for pn, p in (("kernel", l.kernel), ("bias", l.bias)):
                ref = P[f"{name}.{j}.{pn}"].grad
                tol = 1e-4 * float(ref.abs().max())
                if (name, j, pn) == ("i", 2, "bias"):
                    # the sum over the items of their gradients, which is zero: a shift of every item by one
                    # vector changes no probability. What is left is the rounding of 151 terms, 151 2^-24 of
                    # their magnitudes in the sum and 2^-18 of them in the terms
                    tol = (151 * 2.0 ** -24 + 2.0 ** -18) * float(gc.abs().sum(0).max())
                assert float((p.grad.double().cpu() - ref).abs().max()) <= tol, (name, j, pn)
    for emb, ref in ((m.user_embedding, gu), (m.item_embedding, gi)):
        ids, rows = emb.sink.gathered()
        got = torch.zeros_like(ref).index_add_(0, ids.cpu(), rows.double().cpu())
        assert float((got - ref).abs().max()) <= 1e-4 * float(ref.abs().max())


def test_no_dropout_keeps_the_towers_and_modes(cuda):
    """tower_dropout = 0 is the model as it was; in eval mode dropout changes nothing."""
    m, w = build(0.0, precision=6), build(0.5, precision=6)
    w.load_state_dict({**w.state_dict(), **m.state_dict()})
    feats = batch(64, 1)
    a = m(feats)
    b = w(feats, training=False)
    w.eval()
    c = w(feats)
    for k in a:
        assert torch.equal(a[k], b[k]) and torch.equal(a[k], c[k])
    assert torch.equal(m.catalog_loss(feats), w.catalog_loss(feats))
    w.train()
    d = w(feats)
    assert not torch.equal(a["user_embedding"], d["user_embedding"])
    # the whole catalogue, the out-of-vocabulary row first
    enc = m.encode_catalog(training=False)
    assert enc.shape == (NI + 1, D)
    one = m({"movie_id": torch.arange(NI + 1, device="cuda")})["item_embedding"]
    assert torch.equal(enc, one)


def test_train_steps(cuda):
    """Steps with the framework's optimizer: finite losses, every parameter moves, equal seeds give equal
    weights."""
    optim = pkg("optim")

    def run():
        m = build(0.2, precision=6)
        emb = {id(e.weight) for e in (m.user_embedding, m.item_embedding)}
        dense = [p for p in m.parameters() if id(p) not in emb]
        opt = optim.Adagrad(dense, [m.user_embedding, m.item_embedding], optim.ExponentialDecay(0.05), clipnorm=1.0)
        before = {k: v.clone() for k, v in m.state_dict().items()}
        losses = []
        for i in range(4):
            for p in dense:
                p.grad = None
            loss = m.catalog_loss(batch(128, i), reduction="mean")
            loss.backward()
            opt.step()
            losses.append(float(loss))
        return losses, before, m.state_dict()

    losses, before, after = run()
    assert all(np.isfinite(losses))
    for k in before:
        assert not torch.equal(before[k], after[k]), k
    losses2, _, after2 = run()
    assert losses == losses2 and all(torch.equal(after[k], after2[k]) for k in after)


def test_in_batch_loss_with_tower_dropout(cuda):
    """The multi-task step with dropping towers: rows of one id differ, so none may share a row's result;
    the in-batch term is the one of the towers' own outputs."""
    models, F = pkg("models"), pkg("functional")
    cfg = pkg("config").ModelConfig(embedding_dim=64, user_tower_dims=[32], item_tower_dims=[32], dnn_dims=[32])
    m = models.MultiTaskModel(cfg, [str(i) for i in range(5)], [str(i) for i in range(6)], {}, device="cuda",
                              tower_dropout=0.5)
    g = torch.Generator().manual_seed(2)
    B = 300
    feats = {"user_id": torch.randint(0, 6, (B,), generator=g).cuda(),
             "movie_id": torch.randint(0, 7, (B,), generator=g).cuda()}
    labels = {"rating": torch.ones(B, device="cuda"), "y_implicit": torch.ones(B, device="cuda")}
    models.set_dropout_seed(m, 1)
    loss, parts = m.compute_loss((feats, labels), training=True, return_parts=True)
    loss.backward()
    models.set_dropout_seed(m, 1)
    out = m.encoder(feats)
    u, c = out["user_embedding"].detach(), out["item_embedding"].detach()
    assert not torch.equal(u[feats["user_id"] == 3][0], u[feats["user_id"] == 3][1])
    s = u.double() @ c.double().T
    want = float((torch.logsumexp(s, 1) - s.diagonal()).sum())
    assert abs(float(parts["retrieval"].detach()) - want) <= 1e-5 * abs(want)
    assert all(bool(p.grad.isfinite().all()) for p in m.encoder.user_tower.parameters())
    # outside training (a validation step, the exported embeddings) no row is dropped, whatever the module's mode
    states = [d.state.clone() for d in m.modules() if isinstance(d, models.Dropout)]
    plain = models.MultiTaskModel(cfg, [str(i) for i in range(5)], [str(i) for i in range(6)], {}, device="cuda")
    plain.load_state_dict({k: v for k, v in m.state_dict().items() if "dropouts" not in k})
    with torch.no_grad():
        want = plain.compute_loss((feats, labels), training=False)
        assert torch.equal(m.compute_loss((feats, labels), training=False), want)
        want = plain.encoder(feats)
        got = pkg("trainer")._embed(m.encoder, feats)
        pred = m((feats, labels), training=False)["user_embedding"]
    assert torch.equal(got["item_embedding"], want["item_embedding"]) and torch.equal(pred, want["user_embedding"])
    assert all(torch.equal(a, d.state) for a, d in
               zip(states, (d for d in m.modules() if isinstance(d, models.Dropout))))
