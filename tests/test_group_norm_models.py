"""Models with group norm (and 8-bit activation checkpoints): structure, refusals, CPU training."""
import pytest
import torch
import torch.nn.functional as F

from pgdist.config import TrainConfig
from pgdist.engine.trainer import Trainer
from pgdist.models import build_model
from pgdist.ops import nn as N


def test_parameters_and_keys():
    m = build_model("mobilenet_v2", 10, norm="group")
    assert sum(p.numel() for p in m.parameters()) == 2236682   # as with BatchNorm: a weight and a bias a channel
    keys = set(m.state_dict())
    assert "features.2.conv.1.1.weight" in keys and "features.2.conv.3.bias" in keys
    assert not any("running" in k or "num_batches" in k for k in keys)
    assert set(build_model("mobilenet_v2", 10, norm="group", act_ckpt="mx8").state_dict()) == keys
    r = build_model("resnet50", 1000, norm="group", act_ckpt="mx8")
    assert sum(p.numel() for p in r.parameters()) == 25557032


def test_the_default_models_are_unchanged():
    assert not any(isinstance(m, (N.GroupNormAct, N.Conv1x1Ckpt8)) for n in ("mobilenet_v2", "resnet50")
                   for m in build_model(n, 10).modules())


@pytest.mark.parametrize("name", ["mobilenet_v2", "resnet50"])
def test_forward_and_backward_on_cpu(name):
    torch.manual_seed(0)
    m = build_model(name, 10, norm="group")
    x = torch.randn(2, 3, 32, 32)
    out = m(x)
    # images are independent of one another: no batch statistics
    assert torch.allclose(m.eval()(x[:1]), m.eval()(x)[:1], atol=1e-5)
    F.cross_entropy(out, torch.tensor([1, 2])).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


def test_refusals():
    for kw in (dict(norm="layer"), dict(act_ckpt="mx8"), dict(norm="group", act_ckpt="int4")):
        for name in ("mobilenet_v2", "resnet50"):
            with pytest.raises(ValueError):
                build_model(name, 10, **kw)
    x = torch.zeros(2, 12, 4, 4)
    for kw in (dict(groups=5), dict(groups=0), dict(groups=3, act="gelu"), dict(groups=3, weight=torch.ones(11))):
        with pytest.raises(ValueError):
            N.group_norm_act(x, **kw)
    with pytest.raises(ValueError):
        N.group_norm_act(torch.zeros(3), 1)
    with pytest.raises(ValueError):
        N.GroupNormAct(5, 12)
    with pytest.raises(ValueError):
        N.conv1x1(x, torch.zeros(4, 12, 3, 3))


def test_native_executors_refuse_group_norm():
    from pgdist.engine.native_step import executor_class
    with pytest.raises(NotImplementedError, match="BatchNorm"):
        executor_class(build_model("mobilenet_v2", 10, norm="group"))


def _cfg(tmp_path, **kw):
    return TrainConfig(**{**dict(data="synthetic", synthetic_train_size=32, synthetic_test_size=16, batch_size=16,
                                 epochs=1, img_size=32, device="cpu", backend="torch", precision="fp32",
                                 augment="torch", save_path=str(tmp_path / "best.pth"), seed=0, norm="group",
                                 act_ckpt="mx8"), **kw})


def test_trainer_runs_and_saves(tmp_path):
    Trainer(_cfg(tmp_path)).fit()
    sd = torch.load(tmp_path / "best.pth", weights_only=True)
    assert not any("running" in k for k in sd)
    from pgdist.serve.predict import Predictor
    import numpy as np
    p = Predictor(str(tmp_path / "best.pth"), device="cpu", img_size=32, norm="group")
    assert abs(p.probs([np.zeros((32, 32, 3), np.uint8)]).sum().item() - 1) < 1e-5


def test_trainer_refuses_the_native_backend(tmp_path, monkeypatch):
    import pgdist.engine.trainer as T
    monkeypatch.setattr(T, "init_distributed", lambda *a, **k: (type("I", (), dict(rank=0, world_size=1))(),
                                                                 torch.device("cuda"), "nccl"))
    with pytest.raises(NotImplementedError, match="group"):
        Trainer(_cfg(tmp_path, device="cuda", backend="hip"))
