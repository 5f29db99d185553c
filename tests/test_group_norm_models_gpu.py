"""Group norm and 8-bit checkpoints through autograd: gradients, layouts, streams, a training run."""
import pytest
import torch
import torch.nn.functional as F

import gn_oracle as O
from pgdist.ops import kernels as K
from pgdist.ops import nn as N

pytestmark = pytest.mark.gpu


def plain(x, groups, w, b, act):
    y = F.group_norm(x, groups, w, b, 1e-5)
    return {"none": lambda v: v, "relu": F.relu, "relu6": F.relu6, "silu": F.silu}[act](y)


def inputs(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (r(*shape) + 0.3).to(dtype), 1 + 0.2 * r(shape[1]), 0.3 * r(shape[1]), r(*shape).to(dtype)


@pytest.mark.parametrize("act", ["none", "relu", "relu6", "silu"])
@pytest.mark.parametrize("layout", ["channels_last", "contiguous", "strided", "rows"])
def test_gradients_of_every_layout(layout, act):
    shape = (3, 24, 40) if layout == "rows" else (3, 24, 10, 14)
    x, w, b, dy = inputs(shape, torch.float32, 1)
    if layout == "channels_last":
        x = x.contiguous(memory_format=torch.channels_last)
    elif layout == "strided":
        x = torch.randn(3, 24, 20, 14, device="cuda")[:, :, ::2]
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = N.group_norm_act(x, 3, w, b, act=act)
    assert y.shape == x.shape
    got = torch.autograd.grad(y, (x, w, b), dy)
    X, W, B_ = (t.detach().double().requires_grad_() for t in (x, w, b))
    want = torch.autograd.grad(plain(X, 3, W, B_, act), (X, W, B_), dy.double())
    for g, t in zip(got, want):
        # a few hundred roundings of 2^-24 of terms as large as the result's largest
        assert g.shape == t.shape and (g.double() - t).abs().max() <= 1e-5 * t.abs().max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_checkpointed_gradients_are_those_of_the_decoded_input(dtype):
    x, w, b, dy = inputs((4, 40, 9, 7), dtype, 2)
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_()
    w, b = w.requires_grad_(), b.requires_grad_()
    y = N.group_norm_act(x, 5, w, b, act="relu", ckpt8=True)
    got = torch.autograd.grad(y, (x, w, b), dy)
    rows = x.detach().movedim(1, -1).reshape(4, 63, 40)
    q, qs = O.pack(rows.reshape(-1, 40))
    (_, mean, rstd), _ = O.fwd(rows, w, b, 4, 63, 40, 5, 1e-5, 1)
    m2, r2 = torch.empty(4, 5, device="cuda"), torch.empty(4, 5, device="cuda")
    K.gn_fwd(rows.contiguous(), w.detach(), b.detach(), torch.empty_like(rows), m2, r2, 4, 63, 40, 5, act=1)
    want, bound = O.bwd(dy.movedim(1, -1).reshape(4, 63, 40), O.unpack(q, qs), w.detach(), b.detach(), m2, r2, 4, 63,
                        40, 5, 1)
    O.within(got[0].movedim(1, -1).reshape(4, 63, 40), want[0], bound[0])
    O.within(got[1], want[1], bound[1])
    O.within(got[2], want[2], bound[2])


@pytest.mark.parametrize("stride", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_conv1x1(dtype, stride):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 24, 12, 10, generator=g, device="cuda").to(dtype).contiguous(memory_format=torch.channels_last)
    w = (0.2 * torch.randn(40, 24, 1, 1, generator=g, device="cuda")).to(dtype)
    b = torch.randn(40, generator=g, device="cuda").to(dtype)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = N.conv1x1(x, w, b, stride)
    dy = torch.randn(y.shape, generator=g, device="cuda").to(dtype)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xs = x.detach()[:, :, ::stride, ::stride].movedim(1, -1).reshape(-1, 24)
    d = dy.movedim(1, -1).reshape(-1, 40).double()
    W = w.detach().view(40, 24).double()
    h = O.half(dtype)
    want = xs.double() @ W.t() + b.detach().double()
    mag = xs.double().abs() @ W.abs().t() + b.detach().double().abs()
    assert ((y.movedim(1, -1).reshape(-1, 40).double() - want).abs() <= 2 * h * mag).all()   # product, then bias
    X = O.unpack(*O.pack(xs))
    want, mag = d.t().contiguous() @ X, d.abs().t().contiguous() @ X.abs()
    assert ((dw.view(40, 24).double() - want).abs() <= h * want.abs() + 400 * O.U * mag).all()
    assert ((db.double() - d.sum(0)).abs() <= h * d.sum(0).abs() + 400 * O.U * d.abs().sum(0)).all()
    full = torch.zeros(4, 12, 10, 24, dtype=torch.float64, device="cuda")
    full[:, ::stride, ::stride] = (d @ W).view(4, 12 // stride, 10 // stride, 24)
    assert ((dx.movedim(1, -1).double() - full).abs() <= 2 * h * full.abs() + 2 * h * full.abs().mean()).all()


def test_conv1x1_with_a_frozen_weight():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(3, 24, 37, 41, generator=g, device="cuda").bfloat16().contiguous(memory_format=torch.channels_last)
    w = torch.randn(20, 24, 1, 1, generator=g, device="cuda").bfloat16()
    b = torch.zeros(20, device="cuda", requires_grad=True)
    y = N.conv1x1(x, w, b)
    dy = torch.randn(y.shape, generator=g, device="cuda").bfloat16()
    db, = torch.autograd.grad(y, b, dy)
    d = dy.movedim(1, -1).reshape(-1, 20).double()
    O.within(db, O.sums(d), (d.shape[0] + 64) * O.U * O.sums(d.abs()))


def test_under_autocast_parameters_keep_their_type():
    m = torch.nn.Sequential(N.Conv1x1Ckpt8(16, 32), N.GroupNormAct(4, 32, "relu6", ckpt8=True),
                            N.Conv1x1Ckpt8(32, 8)).cuda()
    x = torch.randn(2, 16, 9, 9, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    assert y.dtype == torch.bfloat16
    y.float().square().mean().backward()
    assert x.grad.dtype == torch.float32
    assert all(p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in m.parameters())
    half = N.GroupNormAct(4, 32, "relu").cuda().bfloat16()
    half(torch.randn(2, 32, 5, 5, device="cuda", dtype=torch.bfloat16)).sum().backward()
    assert half.weight.grad.dtype == torch.bfloat16


def test_nothing_is_kept_where_no_gradient_is_wanted():
    x = torch.randn(8, 64, 32, 32, device="cuda", dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
    m = N.GroupNormAct(8, 64, "relu", ckpt8=True).cuda()
    with torch.no_grad():
        a = m(x)
    b = m(x)
    assert torch.equal(a, b) and not a.requires_grad and b.requires_grad
    m.requires_grad_(False)
    xg = x.clone().requires_grad_()
    m(xg).sum().backward()
    assert xg.grad is not None and m.weight.grad is None


def test_on_another_stream():
    x, w, b, dy = inputs((4, 32, 40, 40), torch.bfloat16, 5)
    x = x.contiguous(memory_format=torch.channels_last)

    def once():
        xs = x.detach().requires_grad_()
        y = N.group_norm_act(xs, 4, w, b, act="silu", ckpt8=True)
        return y.detach(), torch.autograd.grad(y, xs, dy)[0]

    want = once()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [once() for _ in range(3)]
    st.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))


def test_under_another_default_type():
    x, w, b, dy = inputs((2, 32, 6, 6), torch.bfloat16, 6)
    conv = (0.1 * torch.randn(16, 32, 1, 1, device="cuda")).bfloat16().requires_grad_()

    def once():
        xs = x.detach().requires_grad_()
        y = N.conv1x1(N.group_norm_act(xs, 4, w.requires_grad_(), b.requires_grad_(), act="relu", ckpt8=True), conv)
        return torch.autograd.grad(y.float().square().sum(), (xs, w, b, conv))

    want = once()
    torch.set_default_dtype(torch.float64)
    try:
        got = once()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_captured_training_step_replays():
    m = torch.nn.Sequential(N.Conv1x1Ckpt8(24, 64), N.GroupNormAct(8, 64, "relu6", ckpt8=True), N.Conv1x1Ckpt8(64, 16),
                            N.GroupNormAct(2, 16, "silu")).cuda().bfloat16().to(memory_format=torch.channels_last)
    g = torch.Generator(device="cuda").manual_seed(8)
    data = [torch.randn(4, 24, 40, 40, generator=g, device="cuda").bfloat16().contiguous(memory_format=torch.channels_last)
            for _ in range(4)]
    x = data[0].clone(memory_format=torch.preserve_format)
    dy = torch.randn(4, 16, 40, 40, generator=g, device="cuda").bfloat16()
    params = list(m.parameters())

    def step():
        return torch.autograd.grad(m(x), params, dy)

    want = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in data:
            x.copy_(d)
            want.append([t.clone() for t in step()])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in (1, 2, 3, 0, 2):
        x.copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        _ = torch.randn(1 << 20, device="cuda").sum().item()   # the program's own work between replays


def test_empty_batches():
    m = N.GroupNormAct(4, 32, "relu", ckpt8=True).cuda()
    x = torch.zeros(0, 32, 5, 5, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = m(x)
    y.sum().backward()
    assert y.shape == x.shape and (m.weight.grad == 0).all()
    c = N.Conv1x1Ckpt8(32, 8).cuda().bfloat16()
    assert c(x.detach()).shape == (0, 8, 5, 5)


@pytest.mark.parametrize("name", ["mobilenet_v2", "resnet50"])
@pytest.mark.parametrize("act_ckpt", ["none", "mx8"])
def test_whole_model_steps(name, act_ckpt):
    from pgdist.models import build_model
    torch.manual_seed(0)
    m = build_model(name, 10, norm="group", act_ckpt=act_ckpt).cuda().to(memory_format=torch.channels_last)
    m.eval()   # no dropout; the norm does not depend on the mode
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(4, 3, 64, 64, generator=g, device="cuda").contiguous(memory_format=torch.channels_last)
    t = torch.tensor([0, 1, 2, 3], device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = m(x)
    F.cross_entropy(out.float(), t).backward()
    grads = {n: p.grad for n, p in m.named_parameters()}
    assert all(torch.isfinite(v).all() for v in grads.values())
    # the same network with plain torch norms and convolutions in fp32
    ref = build_model(name, 10, norm="group").cuda()
    ref.load_state_dict(m.state_dict())
    ref.eval()
    for mod in ref.modules():
        if isinstance(mod, N.GroupNormAct):
            mod.forward = lambda v, mod=mod: plain(v, mod.num_groups, mod.weight, mod.bias, mod.act)
    want = ref(x)
    F.cross_entropy(want, t).backward()
    assert F.cosine_similarity(out.float().flatten(), want.flatten(), dim=0) > 0.99
    last = "classifier.1.weight" if name == "mobilenet_v2" else "fc.weight"
    assert F.cosine_similarity(grads[last].flatten(), dict(ref.named_parameters())[last].grad.flatten(), dim=0) > 0.95


def test_trainer_on_the_gpu(tmp_path):
    from pgdist.config import TrainConfig
    from pgdist.engine.trainer import Trainer
    cfg = TrainConfig(data="synthetic", synthetic_train_size=64, synthetic_test_size=32, batch_size=32, epochs=1,
                      img_size=64, device="cuda", augment="torch", save_path=str(tmp_path / "b.pth"), seed=0,
                      norm="group", act_ckpt="mx8")
    tr = Trainer(cfg)
    assert tr.backend == "torch"
    hist = tr.fit()
    assert hist[0]["train_images"] == 64 and hist[0]["train_loss"] == hist[0]["train_loss"]
