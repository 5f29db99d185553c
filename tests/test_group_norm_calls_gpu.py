"""Group norm and 8-bit checkpoints as programs call them: in-place code behind them, evaluation, odd arguments,
the ends of their ranges."""
import pytest
import torch
import torch.nn.functional as F

import gn_oracle as O
from pgdist.ops import kernels as K
from pgdist.ops import nn as N

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("op,layout", [(op, layout) for op in ("norm", "norm_ckpt8", "conv")
                                       for layout in ("channels_last", "contiguous", "rows")
                                       if (op, layout) != ("conv", "rows")])
def test_in_place_code_behind_an_output(op, layout):
    """relu_ and += on an output give the bits and gradients that the same code gives out of place."""
    shape = (3, 32, 50) if layout == "rows" else (3, 32, 9, 7)
    x = randn(*shape).to(BF)
    if layout == "channels_last":
        x = x.contiguous(memory_format=torch.channels_last)
    w, b, conv = 1 + 0.1 * randn(32, seed=1), randn(32, seed=2), (0.2 * randn(32, 32, 1, 1, seed=3)).to(BF)
    dy = randn(*shape, seed=4).to(BF)

    def run(f):
        leaves = [t.clone().requires_grad_() for t in ((x, conv) if op == "conv" else (x, w, b))]
        if op == "conv":
            y = N.conv1x1(*leaves)
        else:
            y = N.group_norm_act(leaves[0], 4, *leaves[1:], ckpt8=op == "norm_ckpt8")
        y = f(y)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    for plain, inside in ((torch.relu, torch.relu_), (lambda y: y + x, lambda y: y.add_(x))):
        assert all(torch.equal(a, c) for a, c in zip(run(inside), run(plain)))


def test_no_checkpoint_is_made_where_no_gradient_is_wanted(monkeypatch):
    made = []
    fwd, pack = K.gn_fwd, K.mx8_pack
    monkeypatch.setattr(K, "gn_fwd", lambda *a, **k: (made.append(("gn_fwd", k["q"] is not None)), fwd(*a, **k)))
    monkeypatch.setattr(K, "mx8_pack", lambda *a, **k: (made.append(("mx8_pack", True)), pack(*a, **k)))
    m = torch.nn.Sequential(N.Conv1x1Ckpt8(32, 64), N.GroupNormAct(8, 64, "relu", ckpt8=True)).cuda().to(BF)
    x = randn(2, 32, 8, 8).to(BF)
    want = m(x)
    assert made == [("mx8_pack", True), ("gn_fwd", True)] and want.requires_grad
    for off in (torch.no_grad, torch.inference_mode):
        made.clear()
        with off():
            got = m(x)
        assert made == [("gn_fwd", False)] and torch.equal(got, want)


@pytest.mark.parametrize("stride", [(1, 1), (2, 1), (1, 3), (2, 2), [3, 2]])
def test_conv1x1_takes_a_stride_of_each_direction(stride):
    x, w = randn(2, 16, 11, 10).to(BF), (0.2 * randn(24, 16, 1, 1, seed=1)).to(BF)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = N.conv1x1(xs, ws, stride=stride)
    sh, sw = stride
    rows = x[:, :, ::sh, ::sw].movedim(1, -1)
    want = rows.double() @ w.view(24, 16).double().t()
    mag = rows.double().abs() @ w.view(24, 16).double().abs().t()
    assert y.shape == (2, 24, -(-11 // sh), -(-10 // sw))
    # one rounding of the product and its sums in fp32
    assert ((y.movedim(1, -1).double() - want).abs() <= O.half(BF) * want.abs() + 32 * O.U * mag).all()
    c = N.Conv1x1Ckpt8(16, 24, stride if isinstance(stride, tuple) else tuple(stride)).cuda().to(BF)
    with torch.no_grad():
        c.weight.copy_(w)
        assert torch.equal(c(x), y)
    dy = randn(*y.shape, seed=2).to(BF)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    d = dy.movedim(1, -1).reshape(-1, 24).double()
    X = O.unpack(*O.pack(rows.reshape(-1, 16)))
    want, mag = d.t().contiguous() @ X, d.abs().t().contiguous() @ X.abs()
    assert ((dw.view(24, 16).double() - want).abs() <= O.half(BF) * want.abs() + 400 * O.U * mag).all()
    hit = torch.zeros(11, 10, dtype=torch.bool, device="cuda")
    hit[::sh, ::sw] = True
    assert (dx[:, :, ~hit] == 0).all() and (dx[:, :, hit] != 0).any(1).all()


@pytest.mark.parametrize("shape", [(2, 2), (4, 1), (1, 4), (1,), (5,), ()])
def test_parameters_of_other_shapes_are_refused(shape):
    x, bad = torch.zeros(2, 4, 5, 5, device="cuda"), torch.ones(shape, device="cuda")
    for kw in (dict(weight=bad), dict(bias=bad)):
        with pytest.raises(ValueError, match="must be"):
            N.group_norm_act(x, 2, **kw)
    with pytest.raises(ValueError, match="must be"):
        N.conv1x1(x.to(BF), torch.zeros(4, 4, 1, 1, dtype=BF, device="cuda"), bad.to(BF))


def test_conv1x1_of_doubles_stays_double_under_autocast():
    """Autocast leaves fp64 alone."""
    x, w = randn(2, 16, 5, 5).double(), randn(8, 16, 1, 1, seed=1).double()
    with torch.autocast("cuda", dtype=BF):
        y = N.conv1x1(x, w)
    want = (x.movedim(1, -1).cpu() @ w.view(8, 16).t().cpu()).movedim(-1, 1)
    assert y.dtype == torch.float64 and (y.cpu() - want).abs().max() <= 1e-13 * 16 * want.abs().max()


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [(2, 49, 24, 3), (3, 7, 30, 5), (1, 196, 576, 72), (8, 1024, 64, 8), (2, 3136, 144, 18),
                                  (7, 3249, 100, 10), (64, 3136, 32, 4), (1, 60001, 96, 12), (8, 784, 625, 25),
                                  (2, 9, 2049, 1), (3, 333, 264, 11)])
def test_the_bits_of_a_call_with_a_checkpoint_without_one(size, dtype):
    B, S, C, G = size
    x, gamma, beta = randn(B, S, C).to(dtype), 1 + 0.1 * randn(C, seed=1), randn(C, seed=2)
    outs = []
    for ck in (True, False):
        y, mean, rstd = torch.empty_like(x), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
        q = torch.empty(B * S, C, dtype=torch.uint8, device="cuda") if ck else None
        qs = torch.empty(B * S, K.mx8_blocks(C), dtype=torch.uint8, device="cuda") if ck else None
        K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=K.GN_SILU, q=q, qs=qs, as_ckpt8=True)
        outs.append((y, mean, rstd))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("grad", ["no_grad", "inference_mode", "frozen"])
def test_evaluation_has_the_bits_of_training(grad):
    m = N.GroupNormAct(8, 64, "relu", ckpt8=True).cuda()
    for seed in range(8):
        x = randn(8, 64, 32, 32, seed=seed).to(BF).contiguous(memory_format=torch.channels_last)
        want = m(x).detach()
        if grad == "frozen":
            got = m.requires_grad_(False)(x)
            m.requires_grad_(True)
        else:
            with getattr(torch, grad)():
                got = m(x)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,last", [(BF, 8), (torch.float16, 11)])
def test_conv1x1_rounds_product_and_bias_once(dtype, last):
    """2^last + 1 takes a bit more than the type has, so rounded by itself it loses the 1; with a bias of 1 the sum
    2^last + 2 is held exactly."""
    x = torch.ones(1, 8, 2, 2, dtype=dtype, device="cuda")
    w = torch.zeros(8, 8, 1, 1, dtype=dtype, device="cuda")
    w[:, 0], w[:, 1] = 2.0 ** last, 1.0
    b = torch.ones(8, dtype=dtype, device="cuda")
    assert (N.conv1x1(x, w, b) == 2 ** last + 2).all()


@pytest.mark.parametrize("size", [(2, 60, 64, 8), (2, 3001, 96, 12), (2, 60001, 96, 12), (1, 9, 2049, 1)])
@pytest.mark.parametrize("act", [0, 1, 2])
def test_infinite_inputs_keep_their_term_of_dbeta(size, act):
    """Without a border dz is dy whatever x is; where the statistics are NaN, z is, and NaN passes."""
    B, S, C, G = size
    x, dy = randn(B, S, C), randn(B, S, C, seed=1).round()   # whole numbers: dbeta is exact
    x[0, S // 2, 3] = float("inf")
    x[B - 1, S // 3, C - 1] = -float("inf")
    dy[0, S // 2, 3] = dy[B - 1, S // 3, C - 1] = 2
    one, zero = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    K.gn_fwd(x, one, zero, y, mean, rstd, B, S, C, G, act=act)
    dx, dgb = torch.empty_like(x), torch.empty(2, C, device="cuda")
    K.gn_bwd(dy, x, one, zero, mean, rstd, dx, dgb, B, S, C, G, act=act)
    cg = C // G
    z = ((x.view(B, S, G, cg).double() - mean.view(B, 1, G, 1)) * rstd.view(B, 1, G, 1).double()).view(B, S, C)
    out = (z <= 0) if act else torch.zeros_like(z, dtype=torch.bool)
    if act == 2:
        out |= z >= 6
    assert torch.isnan(z[0, :, 3]).all() and torch.isnan(z[B - 1, :, C - 1]).all()
    assert torch.equal(dgb[1].double(), torch.where(out, 0.0, dy.double()).sum((0, 1)))


def test_many_images_of_wide_groups():
    """More (image, channel) pairs than one launch has workgroups for."""
    B, S, C, G = 2050, 2, 8200, 1
    x, dy = randn(B, S, C).to(BF), randn(B, S, C, seed=1).to(BF)
    gamma, beta = 1 + 0.1 * randn(C, seed=2), randn(C, seed=3)
    y, mean, rstd = torch.empty_like(x), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=1)
    want, bound = O.fwd(x, gamma, beta, B, S, C, G, 1e-5, 1)
    for got, w, b in zip((y, mean, rstd), want, bound):
        O.within(got, w, b)
    dx, dgb = torch.full_like(x, float("nan")), torch.full((2, C), float("nan"), device="cuda")
    K.gn_bwd(dy, x, gamma, beta, mean, rstd, dx, dgb, B, S, C, G, act=1)
    want, bound = O.bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, 1)
    for got, w, b in zip((dx, dgb[0], dgb[1]), want, bound):
        O.within(got, w, b)


@pytest.mark.parametrize("ck", [False, True])
def test_more_images_than_one_launch_has_workgroups_for(ck):
    """The images on both sides of the first launch's end, and the last, as they come out alone."""
    B, S, C, G = (1 << 26) + 70, 1, 8, 1
    x, dy = torch.ones(B, S, C, dtype=BF, device="cuda"), torch.zeros(B, S, C, dtype=BF, device="cuda")
    parts = [slice(0, 64), slice((1 << 26) - 80, (1 << 26) + 6), slice(B - 64, B)]
    for i, p in enumerate(parts):
        n = p.stop - p.start
        x[p], dy[p] = randn(n, S, C, seed=i).to(BF), randn(n, S, C, seed=9 + i).round().to(BF)
    y, dx = torch.full_like(x, 7), torch.full_like(x, 7)
    mean, rstd, dgb = torch.full((B, G), 7.0, device="cuda"), torch.full((B, G), 7.0, device="cuda"), torch.empty(2, C, device="cuda")
    q = torch.zeros(B, C, dtype=torch.uint8, device="cuda") if ck else None
    qs = torch.zeros(B, 1, dtype=torch.uint8, device="cuda") if ck else None
    K.gn_fwd(x, None, None, y, mean, rstd, B, S, C, G, q=q, qs=qs)
    K.gn_bwd(dy, None if ck else x, None, None, mean, rstd, dx, dgb, B, S, C, G, q=q, qs=qs)
    for p in parts:
        n = p.stop - p.start
        want = [torch.empty_like(t[p]) for t in (y, mean, rstd)]
        wq = [torch.empty_like(t[p]) for t in (q, qs)] if ck else [None, None]
        K.gn_fwd(x[p].clone(), None, None, *want, n, S, C, G, q=wq[0], qs=wq[1])
        wdx = torch.empty_like(x[p])
        K.gn_bwd(dy[p].clone(), None if ck else x[p].clone(), None, None, *want[1:], wdx, None, n, S, C, G, q=wq[0], qs=wq[1])
        assert all(torch.equal(t[p], w) for t, w in zip((y, mean, rstd, dx), (*want, wdx)))
        assert not ck or (torch.equal(q[p], wq[0]) and torch.equal(qs[p], wq[1]))
    assert bool((mean[64:parts[1].start] == 1).all()) and bool((dx[64:parts[1].start] == 0).all())
    assert torch.equal(dgb[1].double(), sum(dy[p].double().sum((0, 1)) for p in parts))   # whole numbers


def test_backward_of_the_most_channels():
    """One row of 2^30 - 8 channels: the first and the last against the oracle."""
    C = (1 << 30) - 8
    G, n = C // 8, 1 << 14
    x, dy = (torch.empty(1, 1, C, dtype=BF, device="cuda").normal_() for _ in range(2))
    mean, rstd = torch.zeros(1, G, device="cuda"), torch.ones(1, G, device="cuda")   # any will do
    dx, dgb = torch.full_like(x, float("nan")), torch.full((2, C), float("nan"), device="cuda")
    K.gn_bwd(dy, x, None, None, mean, rstd, dx, dgb, 1, 1, C, G, act=1)
    for p, g in ((slice(0, n), slice(0, n // 8)), (slice(C - n, C), slice(G - n // 8, G))):
        want, bound = O.bwd(dy[..., p].contiguous(), x[..., p].contiguous(), None, None, mean[:, g], rstd[:, g], 1, 1, n, n // 8, 1)
        for got, w, b in zip((dx[..., p], dgb[0, p], dgb[1, p]), want, bound):
            O.within(got, w, b)
    for t in (*dx.view(-1).split(1 << 26), *dgb.view(-1).split(1 << 26)):
        assert bool(torch.isfinite(t).all())


def test_pack_of_more_rows_than_one_launch_has_workgroups_for():
    M = (1 << 29) + 37
    x = torch.full((M, 1), 3.0, dtype=BF, device="cuda")
    x[-64:, 0] = randn(64).to(BF)
    q, qs = torch.zeros(M, 1, dtype=torch.uint8, device="cuda"), torch.zeros(M, 1, dtype=torch.uint8, device="cuda")
    K.mx8_pack(x, q, qs, M, 1)
    wq, ws = O.pack(x[-100:])
    assert torch.equal(q[-100:], wq) and torch.equal(qs[-100:], ws)
    assert bool((q[:-64] == wq[0]).all()) and bool((qs[:-64] == ws[0]).all())


def test_wgrad_of_the_most_rows():
    """2^31 - 1 rows, ones but for a few: every sum is a whole number below 2^24 until the splits are joined."""
    M = (1 << 31) - 1
    dy = torch.zeros(M, 1, dtype=BF, device="cuda")
    q, qs = torch.full((M, 1), 0x38, dtype=torch.uint8, device="cuda"), torch.full((M, 1), 127, dtype=torch.uint8, device="cuda")
    at = torch.tensor([0, 63, 64, 12345678, (1 << 30) + 5, M - 2, M - 1], device="cuda")   # 0x38 is 1.0
    dy[at, 0] = torch.arange(1, 8, device="cuda").to(BF)
    dw, db = torch.empty(1, 1, device="cuda"), torch.empty(1, device="cuda")
    K.mx8_wgrad(dy, q, qs, dw, M, 1, 1, db=db)
    assert dw.item() == 28 and db.item() == 28


SOLO, HELD, STAGED, WIDE = range(4)


def both_passes(size, dtype, act, ck_fwd, seed=0):
    """Forward, and backward from x and (ck_fwd) from the checkpoint, against the oracle."""
    B, S, C, G = size
    x, dy = randn(B, S, C, seed=seed).to(dtype), randn(B, S, C, seed=seed + 1).to(dtype)
    gamma, beta = 1 + 0.2 * randn(C, seed=seed + 2), 0.3 * randn(C, seed=seed + 3)
    y, mean, rstd = torch.full_like(x, float("nan")), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    q = torch.zeros(B * S, C, dtype=torch.uint8, device="cuda") if ck_fwd else None
    qs = torch.zeros(B * S, K.mx8_blocks(C), dtype=torch.uint8, device="cuda") if ck_fwd else None
    K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=act, q=q, qs=qs)
    want, bound = O.fwd(x, gamma, beta, B, S, C, G, 1e-5, act)
    for got, w, b in zip((y, mean, rstd), want, bound):
        O.within(got, w, b)
    if ck_fwd:
        wq, ws = O.pack(x.view(B * S, C))
        assert torch.equal(q, wq) and torch.equal(qs, ws)
    for ck in (False, True) if ck_fwd else (False,):
        dx, dgb = torch.full_like(x, float("nan")), torch.full((2, C), float("nan"), device="cuda")
        K.gn_bwd(dy, None if ck else x, gamma, beta, mean, rstd, dx, dgb, B, S, C, G, act=act, q=q if ck else None,
                 qs=qs if ck else None)
        want, bound = O.bwd(dy, O.unpack(q, qs) if ck else x, gamma, beta, mean, rstd, B, S, C, G, act)
        for got, w, b in zip((dx, dgb[0], dgb[1]), want, bound):
            O.within(got, w, b)


@pytest.mark.parametrize("size,dtype,ck,forms", [
    ((2, 6001, 96, 12), BF, False, (HELD, HELD)), ((7, 3249, 100, 10), torch.float32, False, (HELD, HELD)),
    ((4, 40001, 96, 12), BF, True, (STAGED, STAGED)), ((3, 50001, 33, 3), torch.float32, False, (STAGED, STAGED)),
    ((2, 60001, 24, 3), torch.float16, True, (STAGED, HELD))])
@pytest.mark.parametrize("act", [2, 3])
def test_a_wait_that_is_given_up_in_every_form(size, dtype, ck, forms, act):
    """Sums that are not waited for are taken from the tensor, held and staged, forward and backward. A lane then adds
    n / 2 values in a row at most; roundings are as often up as down, so they add as a random walk, to sqrt(n / 2) u / 3,
    which the oracle's (n / 64 + 32) u is six times of at least."""
    lib, dt = K.lib(), {BF: 0, torch.float16: 1, torch.float32: 2}[dtype]
    assert (lib.gn_form(dt, *size, ck, False, act), lib.gn_form(dt, *size, ck, True, act)) == forms
    try:
        lib.gn_set_wait(-1)
        both_passes(size, dtype, act, ck)
    finally:
        lib.gn_set_wait(1 << 16)


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("size,ck", [((3, 400, 2048, 32), True), ((2, 784, 1920, 240), True), ((2, 300, 4096, 32), True),
                                     ((2, 784, 625, 25), True), ((2, 600, 663, 39), True), ((2, 600, 663, 39), False),
                                     ((2, 784, 1280, 160), True)])
def test_wide_rows_of_long_maps(size, ck, dtype):
    """2048 channels in 32 groups, and rows whose checkpoint blocks or sums do not fit one workgroup."""
    both_passes(size, dtype, 1, ck, seed=20)


@pytest.mark.parametrize("act_ckpt", ["none", "mx8"])
@pytest.mark.parametrize("name", ["mobilenet_v2", "resnet50"])
def test_every_layer_of_a_model(name, act_ckpt):
    """A training step under autocast: each norm's and each checkpointed 1x1 convolution's output and gradients against
    the oracle on the operands that it had there. (Whole models are no measure: one relu that falls to the other side
    moves gradients by a hundredth, in torch's own fp32 norms too.)"""
    from pgdist.models import build_model
    torch.manual_seed(0)
    m = build_model(name, 10, norm="group", act_ckpt=act_ckpt).cuda().eval()
    seen = []

    def look(mod, args, y):
        io = dict(mod=mod, x=args[0].detach(), y=y.detach().clone())   # the program may write into y
        args[0].register_hook(lambda g: io.setdefault("dx", g)) if args[0].requires_grad else None
        y.register_hook(lambda g: io.setdefault("dy", g))
        seen.append(io)

    for mod in m.modules():
        if isinstance(mod, (N.GroupNormAct, N.Conv1x1Ckpt8)):
            mod.register_forward_hook(look)
    x = randn(4, 3, 64, 64).contiguous(memory_format=torch.channels_last)
    with torch.autocast("cuda", dtype=BF):
        out = m(x)
    F.cross_entropy(out.float(), torch.tensor([0, 1, 2, 3], device="cuda")).backward()
    assert len(seen) == sum(isinstance(mod, (N.GroupNormAct, N.Conv1x1Ckpt8)) for mod in m.modules()) > 50
    for io in seen:
        mod, (B, C) = io["mod"], io["x"].shape[:2]
        S = io["x"][0, 0].numel()
        rows = lambda t: t.movedim(1, -1).contiguous()  # noqa: E731
        if isinstance(mod, N.GroupNormAct):
            G, act = mod.num_groups, N.ACTS[mod.act]
            xr, w, b = rows(io["x"]).view(B, S, C), mod.weight.detach(), mod.bias.detach()
            y, mean, rstd = torch.empty_like(xr), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
            K.gn_fwd(xr, w, b, y, mean, rstd, B, S, C, G, eps=mod.eps, act=act, as_ckpt8=mod.ckpt8)
            assert torch.equal(rows(io["y"]).view(B, S, C), y)
            want, bound = O.fwd(xr, w, b, B, S, C, G, mod.eps, act)
            O.within(y, want[0], bound[0])
            v = O.unpack(*O.pack(xr.view(B * S, C))) if mod.ckpt8 else xr
            want, bound = O.bwd(rows(io["dy"]).view(B, S, C), v, w, b, mean, rstd, B, S, C, G, act)
            O.within(rows(io["dx"]).view(B, S, C), want[0], bound[0])
            O.within(mod.weight.grad, want[1], bound[1])
            O.within(mod.bias.grad, want[2], bound[2])
        else:
            assert mod.bias is None
            xr = rows(io["x"].to(BF)[:, :, ::mod.stride[0], ::mod.stride[1]]).view(-1, C)
            d, w, M = rows(io["dy"]).view(len(xr), -1).double(), mod.weight.detach().view(-1, C).to(BF).double(), len(xr)
            y = rows(io["y"]).view(M, -1)
            want, mag = xr.double() @ w.t(), xr.double().abs() @ w.abs().t()
            O.within(y, want, O.half(BF) * want.abs() + (C + 1) * O.U * mag)
            X = O.unpack(*O.pack(xr))
            want, mag = d.t().contiguous() @ X, d.abs().t().contiguous() @ X.abs()
            O.within(mod.weight.grad.view(-1, C), want, (M + 64) * O.U * mag)
