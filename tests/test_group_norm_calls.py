"""Group norm and 8-bit checkpoints as programs call them, without a GPU: arguments, checkpoints of models, plans."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.nn.functional as F

from mp_util import free_port, run_ranks
from pgdist.ops import nn as N


@pytest.mark.parametrize("stride", [1, 3, (2,), (1, 1), (2, 1), (1, 3), [3, 2]])
def test_conv1x1_takes_a_stride_of_each_direction(stride):
    x, w, b = torch.randn(2, 4, 11, 10), torch.randn(3, 4, 1, 1), torch.randn(3)
    want = F.conv2d(x, w, b, stride)
    assert torch.equal(N.conv1x1(x, w, b, stride), want)
    m = N.Conv1x1Ckpt8(4, 3, stride, bias=True)
    m.load_state_dict(dict(weight=w, bias=b))
    assert torch.equal(m(x), want)


@pytest.mark.parametrize("stride", [0, -1, (2, 0), (1, 2, 3), ()])
def test_conv1x1_refuses_other_strides(stride):
    with pytest.raises(ValueError, match="stride"):
        N.conv1x1(torch.zeros(2, 4, 5, 5), torch.zeros(3, 4, 1, 1), stride=stride)


@pytest.mark.parametrize("shape", [(2, 2), (4, 1), (1, 4), (1,), (5,), ()])
def test_parameters_of_other_shapes_are_refused(shape):
    """Not only of other counts: their gradients would have another shape than they have."""
    x, bad = torch.zeros(2, 4, 5, 5), torch.ones(shape)
    for kw in (dict(weight=bad), dict(bias=bad)):
        with pytest.raises(ValueError, match="must be"):
            N.group_norm_act(x, 2, **kw)
    for dt in (torch.float32, torch.bfloat16):
        with pytest.raises(ValueError, match="must be"):
            N.conv1x1(x.to(dt), torch.zeros(4, 4, 1, 1, dtype=dt), bad.to(dt))


def test_sizes_past_the_grid_are_refused():
    """Tiles that wait for one another come in one launch; the runtime would take 2^32 work-items and more for fewer."""
    from pgdist.ops import kernels as K
    for bwd in (False, True):
        with pytest.raises(ValueError, match="32-bit grid"):
            K.gn_workspace(1 << 24, 3136, 64, 8, torch.bfloat16, bwd)
        assert K.gn_workspace(1 << 27, 1, 8, 1, torch.bfloat16, bwd) >= 0   # images of their own: several launches


@pytest.mark.parametrize("C", [1 << 30, (1 << 31) - 1, 1 << 31])
def test_checkpoints_of_2_30_channels_and_more_are_refused(C):
    """Their block counts pass 32 bits from 2^31 - 31 on."""
    from pgdist.ops import kernels as K
    x, q = torch.empty(0, dtype=torch.bfloat16), torch.empty(0, dtype=torch.uint8)
    with pytest.raises(ValueError, match="below 2\\^30"):
        K.mx8_pack(x, q, q, 0, C)
    with pytest.raises(ValueError, match="below 2\\^30"):
        K.mx8_unpack(q, q, x, 0, C)


def test_wgrad_plans_for_the_most_rows():
    from pgdist.ops import kernels as K
    for M in ((1 << 31) - 64, (1 << 31) - 63, (1 << 31) - 1):
        # 512 splits of 2^22 rows, each of 8 x 8 products and 8 sums
        assert K.mx8_wgrad_workspace(M, 8, 8) == 512 * (8 * 8 + 8)


@pytest.mark.parametrize("M,N,Kd", [(20000, 1 << 16, 1 << 16), (100, 1 << 19, 1 << 19), (1, (1 << 31) - 1, 1), (1, 1, (1 << 31) - 1),
                                    (1, (1 << 31) - 1, (1 << 31) - 1)])
def test_wgrad_refuses_grids_that_would_not_run_whole(M, N, Kd):
    from pgdist.ops import kernels as K
    with pytest.raises(ValueError, match="too large"):
        K.mx8_wgrad_workspace(M, N, Kd)


def test_pretrained_weights_of_the_other_norm_are_refused(tmp_path):
    """With another number of classes too, where the head's weights are left out."""
    from pgdist.models import build_model
    path = str(tmp_path / "w.pth")
    for name in ("mobilenet_v2", "resnet50"):
        for saved, wanted in (("batch", "group"), ("group", "batch")):
            torch.save(build_model(name, 10, norm=saved).state_dict(), path)
            for classes in (10, 7):
                with pytest.raises((ValueError, RuntimeError)):
                    build_model(name, classes, pretrained=path, norm=wanted)
                m = build_model(name, classes, pretrained=path, norm=saved)
                sd = torch.load(path, weights_only=True)
                assert all(torch.equal(v, sd[k]) for k, v in m.state_dict().items() if sd[k].shape == v.shape
                           and not k.startswith(("fc.", "classifier.")))


def test_trainer_refuses_fp8_with_group_norm():
    """It would train in fp32 on the torch backend without a word."""
    from pgdist.config import TrainConfig
    from pgdist.engine.trainer import Trainer
    with pytest.raises(NotImplementedError, match="fp8"):
        Trainer(TrainConfig(data="synthetic", synthetic_train_size=8, synthetic_test_size=8, batch_size=8, img_size=32,
                            device="cpu", norm="group", precision="fp8"))


def test_forms_of_group_norm():
    """SOLO, HELD, STAGED, WIDE by size, type and direction (bf16, fp16, fp32 are 0, 1, 2)."""
    from pgdist.ops import kernels as K
    form = K.lib().gn_form
    assert form(0, 1, 49, 1280, 160, False, False, 0) == form(0, 1, 49, 1280, 160, False, True, 0) == 0
    assert form(2, 7, 3249, 100, 10, False, False, 0) == form(0, 96, 784, 192, 24, True, True, 0) == 1
    assert form(0, 128, 3136, 144, 18, True, False, 0) == form(0, 128, 12544, 96, 12, False, True, 0) == 2
    assert form(0, 2, 9, 2049, 1, False, False, 0) == form(0, 2050, 2, 8200, 1, False, True, 0) == 3


def _train_two_ranks(rank, world, port, tmp, bn_sync, q):
    import pgdist  # noqa: F401
    from pgdist.config import TrainConfig
    from pgdist.engine.trainer import Trainer
    from pgdist.parallel.bootstrap import DistInfo
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    info = DistInfo(rank=rank, world_size=world, local_rank=rank, local_world_size=world, master_port=port)
    tr = Trainer(TrainConfig(data="synthetic", synthetic_train_size=32, synthetic_test_size=16, batch_size=8, epochs=1,
                             img_size=32, device="cpu", backend="torch", precision="fp32", augment="none", norm="group",
                             act_ckpt="mx8", save_path=os.path.join(tmp, "b.pth"), log_format="ddp", seed=42,
                             bn_sync=bn_sync), info=info)
    tr.fit()
    q.put(("ok", rank, tr.replicas_ok, tr.history[-1]["train_images"]))
    dist.destroy_process_group()


@pytest.mark.parametrize("bn_sync", ["eval", "broadcast"])
def test_two_ranks_train_without_batch_statistics(tmp_path, bn_sync):
    """There are no buffers to broadcast or compare."""
    for _, rank, ok, n in run_ranks(_train_two_ranks, 2, (2, free_port(), str(tmp_path), bn_sync), expect=2, timeout=300):
        assert ok == (True, True) and n == 32
