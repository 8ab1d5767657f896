"""The catalogue softmax and dropout where no GPU is needed: refusals before any launch, workspace
queries, the modules' configuration."""
import pytest
import torch

from conftest import pkg

A = 4096  # a 16-byte aligned address that no call below dereferences


def fwd(N=4, V=8, D=16, dtype=0, scale=1.0, want=3, keep=1 << 30, ws=1 << 30, x=A, w=A, labels=A):
    pkg("_native").call("rs_catalog_softmax_fwd", x, w, labels, None, N, V, D, dtype, scale, -100, 0, want, A, A, A, A,
                        keep, A, ws, None)


def test_cpu_tensors_are_refused():
    F = pkg("functional")
    x, y = torch.zeros((4, 8)), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.catalog_softmax_fwd(x, x, y)
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.catalog_softmax_loss(x, x, y)
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.dropout_apply(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.dropout_ticket(torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("bad,match", [
    (dict(N=-1), "bad sizes"), (dict(V=0), "bad sizes"), (dict(D=0), "bad sizes"), (dict(N=1 << 26), "2\\^26"),
    (dict(V=1 << 29), "2\\^29"), (dict(N=1 << 25, D=256), "2\\^33"), (dict(D=257), "above 256"),
    (dict(dtype=7), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(want=4), "flags"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(labels=None), "null"), (dict(x=A + 4), "aligned"), (dict(w=A + 8), "aligned"), (dict(keep=64), "keep"),
    (dict(ws=64), "workspace")])
def test_forward_refusals(bad, match):
    with pytest.raises(pkg("_native").NativeError, match=match):
        fwd(**bad)


def test_backward_refusals():
    N = pkg("_native")

    def bwd(want=3, keep=1 << 30, ws=1 << 30, dx=A, dw=A, w=A):
        N.call("rs_catalog_softmax_bwd", w, 4, 8, 16, 0, 1.0, want, None, A, keep, dx, dw, A, ws, None)

    for bad, match in ((dict(want=2), "dX needs"), (dict(want=1), "dW needs"), (dict(w=None), "null"),
                       (dict(dw=A + 2), "aligned"), (dict(keep=64), "keep")):
        with pytest.raises(N.NativeError, match=match):
            bwd(**bad)


def test_dropout_refusals():
    N = pkg("_native")
    for args, match in (((A, -1, 0, 0.5, A, A), "bad size"), ((A, 8, 9, 0.5, A, A), "dtype"),
                        ((A, 1 << 35, 1, 0.5, A, A), "2.35"), ((A, 8, 0, 1.0, A, A), "rate"),
                        ((A, 8, 0, -0.5, A, A), "rate"),
                        ((A, 8, 0, float("nan"), A, A), "rate"), ((A, 8, 0, 1 - 2.0 ** -40, A, A), "keeps no element"),
                        ((None, 8, 0, 0.5, A, A), "null")):
        with pytest.raises(N.NativeError, match=match):
            N.call("rs_dropout", *args, None)
    N.call("rs_dropout", None, 0, 0, 0.5, None, None, None)   # nothing to do
    with pytest.raises(N.NativeError, match="shared"):
        N.call("rs_dropout_ticket", A, A, None)


def test_workspace_queries():
    q = pkg("_native").query
    for dt in (0, 1):
        for n, v, d in ((0, 1, 1), (1, 1, 1), (1000, 50_000, 96), (65_536, 1_000_000, 256)):
            none = q("rs_catalog_softmax_keep_bytes", n, v, d, dt, 0)
            both = q("rs_catalog_softmax_keep_bytes", n, v, d, dt, 3)
            assert both >= none + 4 * n * d
            assert q("rs_catalog_softmax_workspace_bytes", n, v, d, dt, 3) > 0
    assert q("rs_catalog_softmax_keep_bytes", 4, 4, 300, 0, 0) == 0   # unsupported width
    # sizes whose grids would pass 2^32 threads
    for n, v, d in ((1 << 26, 4, 1), (4, 1 << 29, 1), (1 << 25, 4, 256)):
        assert q("rs_catalog_softmax_keep_bytes", n, v, d, 1, 0) == 0
        assert q("rs_catalog_softmax_keep_bytes", n - 1 if n > v else n, v - 1 if v > n else v, d, 1, 0) > 0
    # the same sizes, other types and gradients: each its own plan
    ask = [(dt, w) for dt in (0, 1) for w in (0, 1, 2, 3)]
    first = [q("rs_catalog_softmax_workspace_bytes", 64, 50_000, 128, dt, w) for dt, w in ask]
    for (dt, w), b in zip(reversed(ask), reversed(first)):
        assert q("rs_catalog_softmax_workspace_bytes", 64, 50_000, 128, dt, w) == b


def test_the_loss_alone_without_gradients(monkeypatch):
    """With gradients disabled no gradient's work is asked for, though the operands require them."""
    F = pkg("functional")
    asked = []

    def fwd(X, W, labels, scale, weights, ignore_index, reduction, want_grad, want_lse):
        asked.append(want_grad)
        st = F.CatalogSoftmaxState(torch.empty(1), X.shape[0], W.shape[0], X.shape[1], X.dtype, scale, 0, 256)
        return torch.zeros(()), torch.zeros(X.shape[0]), None, st

    monkeypatch.setattr(F, "_catalog_fwd", fwd)
    x, w = torch.zeros((3, 8)), torch.zeros((5, 8), requires_grad=True)
    y = torch.zeros(3, dtype=torch.int64)
    loss, _ = F.catalog_softmax_loss(x, w, y)
    assert loss.requires_grad and asked == [(False, True)]
    with torch.no_grad():
        loss, _ = F.catalog_softmax_loss(x, w, y, weights=torch.ones(3, requires_grad=True))
    assert not loss.requires_grad and asked[1] is False


def test_modules():
    models, cfgm = pkg("models"), pkg("config")
    for rate in (-0.1, 1.0):
        with pytest.raises(ValueError, match="rate"):
            models.Dropout(rate, device="cpu")
    drop = models.Dropout(0.3, seed=4, device="cpu").eval()
    x = torch.ones((2, 3))
    assert drop(x) is x and drop.state.tolist() == [4, 0] and models.Dropout(0.0, device="cpu")(x) is x
    plain = models.Tower(8, [16, 8], 4, device="cpu")
    wet = models.Tower(8, [16, 8], 4, device="cpu", dropout_rate=0.5)
    assert plain.dropouts is None and not plain.drops() and wet.drops() and not wet.eval().drops()
    assert set(wet.state_dict()) - set(plain.state_dict()) == {"dropouts.0.state", "dropouts.1.state"}
    assert len({tuple(d.state.tolist()) for d in wet.dropouts}) == 2
    models.set_dropout_seed(wet, 9)
    assert [d.state.tolist() for d in wet.dropouts] == [[9, 0], [9 + 7919, 0]]
    cfg = cfgm.ModelConfig(embedding_dim=16, user_tower_dims=[8], item_tower_dims=[8])
    enc = models.MultiTowerModel(cfg, ["a"], ["b"], {}, device="cpu")
    assert "tower_dropout" not in enc.get_config() and enc.user_tower.dropouts is None
    wet = models.MultiTowerModel(cfg, ["a"], ["b"], {}, device="cpu", tower_dropout=0.25)
    again = models.MultiTowerModel.from_config(wet.get_config(), device="cpu")
    assert again.tower_dropout == 0.25 and len(again.item_tower.dropouts) == 1


def test_multi_task_config_keeps_the_tower_dropout():
    """A model rebuilt from its configuration drops alike and takes the original's state; without dropout the
    configuration holds what it held."""
    models, cfgm = pkg("models"), pkg("config")
    cfg = cfgm.ModelConfig(embedding_dim=16, user_tower_dims=[8], item_tower_dims=[8], dnn_dims=[8])
    wet = models.MultiTaskModel(cfg, ["a"], ["b"], {}, class_weights={0: 0.5, 1: 2.0}, device="cpu", tower_dropout=0.25)
    again = models.MultiTaskModel.from_config(wet.get_config(), device="cpu")
    assert again.encoder.tower_dropout == 0.25 and again.class_weights == {0: 0.5, 1: 2.0}
    again.load_state_dict(wet.state_dict())
    plain = models.MultiTaskModel(cfg, ["a"], ["b"], {}, device="cpu")
    assert set(plain.get_config()) == {"config", "user_vocab", "item_vocab", "feature_specs", "class_weights"}


def test_a_model_with_dropout_is_served(tmp_path, monkeypatch):
    """The artefacts of a model with tower dropout, as the trainer writes them and as its checkpoint holds them, load
    into the services, whose models have none."""
    models, cfgm, trainer = pkg("models"), pkg("config"), pkg("trainer")
    cfg = cfgm.ModelConfig(embedding_dim=16, user_tower_dims=[8], item_tower_dims=[8], dnn_dims=[8])
    users, items = ["a", "b"], ["c", "d", "e"]
    wet = models.MultiTaskModel(cfg, users, items, {}, device="cpu", tower_dropout=0.25)
    tr = trainer.ProductionTrainer.__new__(trainer.ProductionTrainer)
    tr.config, tr.output_dir = cfg, tmp_path
    tr._save_artifacts(wet, {"user_vocab": users, "item_vocab": items})
    torch.save(wet.state_dict(), tmp_path / "best_model.pt")
    (tmp_path / "item_map.json").write_text('{"0": "c", "1": "d", "2": "e"}')
    torch.save(torch.eye(3, 16), tmp_path / "item_index.pt")
    cpu = torch.device("cpu")
    svc = pkg("serving").RecommendationService(str(tmp_path), cpu)
    svc.load()
    ms = pkg("model_service").RecommendationService(str(tmp_path), cpu)
    monkeypatch.setattr(ms, "_precompute_item_embeddings", lambda: None)   # (GPU kernels)
    ms.load_model()
    for enc in (svc.encoder_model, ms.model):
        want = wet.encoder.state_dict()
        for k, v in enc.state_dict().items():
            assert torch.equal(v, want[k]), k
    # an encoder.pt that holds the generators too
    torch.save(wet.encoder.state_dict(), tmp_path / "encoder.pt")
    svc.load()
    # the generators stay in the model's own state
    assert "encoder.user_tower.dropouts.0.state" in wet.state_dict()


def test_rows_are_not_grouped_by_id_where_the_towers_drop(monkeypatch):
    """compute_loss takes `training` as the towers do: None is the module's mode."""
    models, cfgm = pkg("models"), pkg("config")
    cfg = cfgm.ModelConfig(embedding_dim=16, user_tower_dims=[8], item_tower_dims=[8], dnn_dims=[8])
    B = 4
    batch = ({"user_id": torch.zeros(B, dtype=torch.int64), "movie_id": torch.ones(B, dtype=torch.int64)},
             {"rating": torch.zeros(B)})
    seen = []

    class Stop(Exception):
        pass

    class Cross:
        @staticmethod
        def apply(u, i, w, b, prec, ids):
            seen[-1] += (ids is not None,)
            raise Stop

    monkeypatch.setattr(models, "RetrievalCrossFn", Cross)
    for rate, grouped in ((0.5, {(True, None): False, (True, True): False, (True, False): True,
                                 (False, None): True, (False, True): False}), (0.0, {(True, None): True, (True, True): True})):
        m = models.MultiTaskModel(cfg, ["a"], ["b"], {}, device="cpu", tower_dropout=rate)
        monkeypatch.setattr(m, "_towers", lambda f, orders=None, training=None: (seen.append((training,)), (None, None))[1])
        for (mode, training), want in grouped.items():
            with pytest.raises(Stop):
                m.train(mode).compute_loss(batch, training=training)
            assert seen[-1] == (training, want), (rate, mode, training)


@pytest.mark.parametrize("rate", [-0.5, 1.0, float("nan")])
def test_towers_refuse_what_dropout_refuses(rate):
    models, cfgm = pkg("models"), pkg("config")
    cfg = cfgm.ModelConfig(embedding_dim=16, user_tower_dims=[8], item_tower_dims=[8], dnn_dims=[8])
    with pytest.raises(ValueError, match="rate"):
        models.Tower(8, [16], 4, device="cpu", dropout_rate=rate)
    with pytest.raises(ValueError, match="rate"):
        models.MultiTowerModel(cfg, ["a"], ["b"], {}, device="cpu", tower_dropout=rate)
    with pytest.raises(ValueError, match="rate"):
        models.MultiTaskModel(cfg, ["a"], ["b"], {}, device="cpu", tower_dropout=rate)


def test_forward_mode_is_refused(monkeypatch):
    """A tangent is refused, with gradients enabled or not (no_grad leaves forward mode on), and never lost."""
    F = pkg("functional")
    from torch.autograd import forward_ad

    def fwd(X, W, labels, scale, weights, ignore_index, reduction, want_grad, want_lse):
        st = F.CatalogSoftmaxState(torch.empty(1), X.shape[0], W.shape[0], X.shape[1], X.dtype, scale, 0, 256)
        return torch.zeros(()), torch.zeros(X.shape[0]), None, st

    monkeypatch.setattr(F, "_catalog_fwd", fwd)
    x, w, a = torch.zeros((3, 8)), torch.zeros((5, 8)), torch.ones(3)
    y = torch.zeros(3, dtype=torch.int64)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            for dual in ("x", "w", "a"):
                t = {"x": x, "w": w, "a": a}
                t[dual] = forward_ad.make_dual(t[dual], torch.ones_like(t[dual]))
                with pytest.raises(NotImplementedError):
                    F.catalog_softmax_loss(t["x"], t["w"], y, weights=t["a"])
            F.catalog_softmax_loss(x, w, y, weights=a)
