"""Group norm + activation (forward, backward, fused checkpoint) against 64-bit oracles."""
import pytest
import torch

import gn_oracle as O
from pgdist.ops import kernels as K

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5

# (B, S, C, G): one value to long maps, odd channels, one group, instance norm, groups that straddle vectors
SIZES = [(1, 1, 1, 1), (1, 1, 8, 1), (2, 3, 8, 2), (3, 7, 30, 5), (2, 49, 24, 3), (2, 100, 33, 3), (2, 65, 16, 16),
         (1, 196, 576, 72), (1, 49, 1280, 160), (2, 49, 2048, 32), (4, 784, 64, 8), (2, 3136, 144, 18),
         (1, 3, 8192, 1), (2, 5, 1000, 1), (1, 12544, 96, 12), (5, 1021, 100, 10), (1, 50176, 4, 2), (130, 9, 40, 5),
         (2, 4097, 12, 1), (1, 257, 17, 17), (1, 40001, 31, 1), (3, 333, 264, 11)]


def make(B, S, C, dt, seed=0, level=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (r(B, S, C) * (0.5 + r(C).abs()) + 0.7 * r(C) + level * r(B, 1, 1)).to(dt)
    return x, 1 + 0.2 * r(C), 0.3 * r(C), r(B, S, C).to(dt)


def call_fwd(x, gamma, beta, B, S, C, G, act=0, ck=False, eps=EPS, ws=None):
    y = torch.full_like(x, float("nan"))
    mean = torch.full((B, G), float("nan"), device="cuda")
    rstd = mean.clone()
    q = torch.zeros(B * S, C, dtype=torch.uint8, device="cuda") if ck else None
    qs = torch.zeros(B * S, K.mx8_blocks(C), dtype=torch.uint8, device="cuda") if ck else None
    K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, eps=eps, act=act, q=q, qs=qs, ws=ws)
    return y, mean, rstd, q, qs


def call_bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, act=0, q=None, qs=None, params=True, ws=None):
    dx = torch.full_like(dy, float("nan"))
    dgb = torch.full((2, C), float("nan"), device="cuda") if params else None
    K.gn_bwd(dy, x, gamma, beta, mean, rstd, dx, dgb, B, S, C, G, act=act, q=q, qs=qs, ws=ws)
    return dx, dgb


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_forward(i, dtype):
    B, S, C, G = SIZES[i]
    act, ck, affine = i % 4, i % 3 != 0, i % 5 != 4
    x, gamma, beta, _ = make(B, S, C, DT[dtype], i)
    if not affine:
        gamma = beta = None
    y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, act, ck)
    want, bound = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)
    for got, w, b in zip((y, mean, rstd), want, bound):
        O.within(got, w, b)
    if ck:
        wq, ws = O.pack(x.view(B * S, C))
        assert torch.equal(qs, ws) and torch.equal(q, wq)


@pytest.mark.parametrize("act", range(4))
@pytest.mark.parametrize("size", [(2, 49, 24, 3), (3, 1021, 100, 10), (2, 3136, 144, 18)])
def test_forward_every_activation(size, act):
    B, S, C, G = size
    x, gamma, beta, _ = make(B, S, C, torch.float32, 5)
    want, bound = O.fwd(x, gamma, 3 * beta, B, S, C, G, EPS, act)
    got = call_fwd(x, gamma, 3 * beta, B, S, C, G, act)
    for k in range(3):
        O.within(got[k], want[k], bound[k])


@pytest.mark.parametrize("ck", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_backward(i, dtype, ck):
    B, S, C, G = SIZES[i]
    act, affine = (i + 1) % 4, i % 5 != 4
    x, gamma, beta, dy = make(B, S, C, DT[dtype], 50 + i)
    if not affine:
        gamma = beta = None
    _, mean, rstd = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)[0]
    mean, rstd = mean.float(), rstd.float()
    q = qs = None
    v = x
    if ck:
        q, qs = O.pack(x.view(B * S, C))
        v, x = O.unpack(q, qs), None
    dx, dgb = call_bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, act, q, qs)
    want, bound = O.bwd(dy, v, gamma, beta, mean, rstd, B, S, C, G, act)
    for got, w, b in zip((dx, dgb[0], dgb[1]), want, bound):
        O.within(got, w, b)
    again, none = call_bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, act, q, qs, params=False)
    assert none is None and torch.equal(again, dx)


@pytest.mark.parametrize("act", range(4))
def test_backward_every_activation(act):
    B, S, C, G = 2, 1021, 100, 10
    x, gamma, beta, dy = make(B, S, C, torch.float32, 9)
    beta = 3 * beta
    _, mean, rstd = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)[0]
    dx, dgb = call_bwd(dy, x, gamma, beta, mean.float(), rstd.float(), B, S, C, G, act)
    want, bound = O.bwd(dy, x, gamma, beta, mean.float(), rstd.float(), B, S, C, G, act)
    for got, w, b in zip((dx, dgb[0], dgb[1]), want, bound):
        O.within(got, w, b)


@pytest.mark.parametrize("act", [0, 3])
def test_backward_against_differences(act):
    """d/dt sum(dy * f(x + t v)) at 0, f evaluated in 64 bits, against <dx, v> (dgamma, dbeta alike).
    The central difference of step h is off by O(h^2) of third derivatives, which are O(10) here:
    1e-8 at h = 1e-5 with 1e-16 / h = 1e-11 of rounding, both far below fp32's own error."""
    B, S, C, G = 2, 37, 24, 3
    x, gamma, beta, dy = make(B, S, C, torch.float32, 3)
    (_, mean, rstd), _ = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)
    dx, dgb = call_bwd(dy, x, gamma, beta, mean.float(), rstd.float(), B, S, C, G, act)
    gen = torch.Generator(device="cuda").manual_seed(1)
    f = lambda a, g, b: (dy.double() * O.fwd(a, g, b, B, S, C, G, EPS, act)[0][0]).sum()  # noqa: E731
    h = 1e-5
    X, g, b = x.double(), gamma.double(), beta.double()
    for k in range(3):
        v = torch.randn((X, g, b)[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        p, m = [X, g, b], [X, g, b]
        p[k], m[k] = p[k] + h * v, m[k] - h * v
        num = ((f(*p) - f(*m)) / (2 * h)).item()
        terms = (dx, dgb[0], dgb[1])[k].double().view_as(v) * v
        assert abs(num - terms.sum().item()) <= 1e-5 * terms.abs().sum().item() + 1e-6


# groups of more vectors than a workgroup has threads; maps of more tiles than wait for one another
FAR_SIZES = [(2, 9, 2049, 1), (1, 5, 4100, 2), (2, 3, 9000, 1), (1, 400000, 32, 4), (1, 300001, 12, 3), (2, 130000, 75, 5)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("i", range(len(FAR_SIZES)))
def test_wide_groups_and_long_maps(i, dtype):
    B, S, C, G = FAR_SIZES[i]
    act = (0, 1, 3, 2, 3, 1)[i]
    x, gamma, beta, dy = make(B, S, C, DT[dtype], 70 + i)
    y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, act, True)
    want, bound = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)
    for got, w, b in zip((y, mean, rstd), want, bound):
        O.within(got, w, b)
    wq, ws = O.pack(x.view(B * S, C))
    assert torch.equal(qs, ws) and torch.equal(q, wq)
    for ck in (False, True):
        v = O.unpack(q, qs) if ck else x
        dx, dgb = call_bwd(dy, None if ck else x, gamma, beta, mean, rstd, B, S, C, G, act, q if ck else None,
                           qs if ck else None)
        want, bound = O.bwd(dy, v, gamma, beta, mean, rstd, B, S, C, G, act)
        for got, w, b in zip((dx, dgb[0], dgb[1]), want, bound):
            O.within(got, w, b)


@pytest.mark.parametrize("size", [(2, 6001, 96, 12), (3, 2001, 33, 3)])
def test_a_wait_that_is_given_up(size):
    """With no polls left, sums that have not come in time are taken from the tensor itself."""
    B, S, C, G = size
    lib = K.lib()
    for dt, act in ((torch.bfloat16, 2), (torch.float32, 3)):
        x, gamma, beta, dy = make(B, S, C, dt, 8)
        try:
            lib.gn_set_wait(-1)
            y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, act, True)
            dx = call_bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, act)[0]
            dxq = call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, act, q, qs)[0]
        finally:
            lib.gn_set_wait(1 << 16)
        want, bound = O.fwd(x, gamma, beta, B, S, C, G, EPS, act)
        for got, w, b in zip((y, mean, rstd), want, bound):
            O.within(got, w, b)
        for got, v in ((dx, x), (dxq, O.unpack(q, qs))):
            want, bound = O.bwd(dy, v, gamma, beta, mean, rstd, B, S, C, G, act)
            O.within(got, want[0], bound[0])


def test_far_mean_keeps_its_variance():
    """mean 1000, deviation 1: the squares are taken about the mean, not as E[x^2] - mean^2."""
    for B, S, C, G in ((1, 196, 32, 4), (1, 60000, 8, 1), (2, 12544, 64, 2)):
        g = torch.Generator(device="cuda").manual_seed(1)
        x = 1000 + torch.randn(B, S, C, generator=g, device="cuda")
        _, mean, rstd, _, _ = call_fwd(x, None, None, B, S, C, G)
        want, bound = O.fwd(x, None, None, B, S, C, G, EPS, 0)
        assert ((rstd.double() - want[2]).abs() <= 1e-4).all()
        O.within(mean, want[1], bound[1])


def test_non_finite_values_stay_in_their_group():
    B, S, C, G = 2, 100, 64, 8
    x, gamma, beta, dy = make(B, S, C, torch.bfloat16, 2)
    clean = call_fwd(x, gamma, beta, B, S, C, G, 1, True)
    bad = x.clone()
    bad[0, 5, 9] = float("nan")
    bad[1, 7, 40] = float("inf")
    y, mean, rstd, q, qs = call_fwd(bad, gamma, beta, B, S, C, G, 1, True)
    hit = torch.zeros(B, S, G, C // G, dtype=torch.bool, device="cuda")
    hit[0, :, 1] = hit[1, :, 5] = True
    hit = hit.view(B, S, C)
    assert torch.isnan(y[0, :, 8:16]).all() and torch.isnan(y[1, :, 40:48]).all()
    assert torch.equal(y[~hit], clean[0][~hit])
    wq, ws = O.pack(bad.view(B * S, C))
    assert torch.equal(qs, ws)
    assert torch.equal(q & 127, wq & 127)   # a NaN's sign says nothing
    dx, dgb = call_bwd(dy, bad, gamma, beta, mean, rstd, B, S, C, G, 1)
    dx0, _ = call_bwd(dy, x, gamma, beta, clean[1], clean[2], B, S, C, G, 1)
    assert torch.isnan(dx[hit]).all() and torch.equal(dx[~hit], dx0[~hit])
    touched = torch.isnan(dgb[0])
    assert touched[8:16].any() and not touched[:8].any() and not touched[16:40].any() and not touched[48:].any()


def test_borders_are_decided_in_64_bits():
    """Values whose z lies within fp32's error of relu's border: the gradient passes where z > 0."""
    B, S, C, G = 1, 512, 8, 1
    mean = torch.tensor([[0.3]], device="cuda")
    rstd = torch.tensor([[1.7]], device="cuda")
    gamma = torch.full((C,), 0.9, device="cuda")
    beta = torch.full((C,), -0.4, device="cuda")
    x0 = 0.3 + 0.4 / (1.7 * 0.9)
    x = (torch.full((B, S, C), x0, device="cuda", dtype=torch.float64).float().view(-1).view(torch.int32)
         + torch.arange(-2048, 2048, device="cuda", dtype=torch.int32)).view(torch.float32).view(B, S, C)
    dy = torch.ones(B, S, C, device="cuda")
    for act, bt in ((1, beta), (2, beta), (2, beta + 6)):
        _, dgb = call_bwd(dy, x, gamma, bt, mean, rstd, B, S, C, G, act)
        z = (x.double() - mean.double()) * rstd.double() * gamma.double() + bt.double()
        want = ((z > 0) & (z < 6)).double() if act == 2 else (z > 0).double()
        assert torch.equal(dgb[1].double(), want.sum((0, 1)))   # whole numbers below 2^24: exact in fp32


def test_empty_sizes():
    for B, S in ((0, 5), (3, 0)):
        x, gamma, beta, dy = make(B, S, 16, torch.bfloat16)
        y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, 16, 2, 1, True)
        assert (mean == 0).all() and torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5))
        dx, dgb = call_bwd(dy, x, gamma, beta, mean, rstd, B, S, 16, 2, 1)
        assert (dgb == 0).all() and dx.numel() == 0


@pytest.mark.parametrize("size", [(2, 49, 24, 3), (3, 6001, 96, 12), (2, 2001, 75, 5)])
def test_same_bits_every_time_and_nothing_written_behind(size):
    B, S, C, G = size
    x, gamma, beta, dy = make(B, S, C, torch.bfloat16, 4)
    n = B * S * C
    first = None
    for _ in range(3):
        buf = [torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        q = torch.full((n + 64,), 9, dtype=torch.uint8, device="cuda")
        ns = B * S * K.mx8_blocks(C)
        qs = torch.full((ns + 64,), 9, dtype=torch.uint8, device="cuda")
        st = torch.full((2, B * G + 64), 5.0, device="cuda")
        dgb = torch.full((2 * C + 64,), 5.0, device="cuda")
        mean, rstd = st[0, :B * G], torch.empty(B * G, device="cuda")
        y, dx = buf[0][:n].view(B, S, C), buf[1][:n].view(B, S, C)
        K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=2, q=q[:n], qs=qs[:ns])
        K.gn_bwd(dy, None, gamma, beta, mean, rstd, dx, dgb[:2 * C].view(2, C), B, S, C, G, act=2, q=q[:n], qs=qs[:ns])
        assert (buf[0][n:] == 7).all() and (buf[1][n:] == 7).all() and (q[n:] == 9).all() and (qs[ns:] == 9).all()
        assert (st[0, B * G:] == 5).all() and (dgb[2 * C:] == 5).all()
        out = (y.clone(), mean.clone(), rstd, q[:n].clone(), qs[:ns].clone(), dx.clone(), dgb[:2 * C].clone())
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize("size", [(2, 49, 64, 8), (2, 12544, 96, 12)])
def test_captured_and_replayed(size):
    B, S, C, G = size
    x, gamma, beta, dy = make(B, S, C, torch.bfloat16, 6)
    ws = [torch.empty(K.gn_workspace(B, S, C, G, x.dtype, b) + 4, device="cuda") for b in (False, True)]
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    q = torch.empty(B * S, C, dtype=torch.uint8, device="cuda")
    qs = torch.empty(B * S, K.mx8_blocks(C), dtype=torch.uint8, device="cuda")
    dgb = torch.empty(2, C, device="cuda")

    def step():
        K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=2, q=q, qs=qs, ws=ws[0])
        K.gn_bwd(dy, None, gamma, beta, mean, rstd, dx, dgb, B, S, C, G, act=2, q=q, qs=qs, ws=ws[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        x.copy_(make(B, S, C, torch.bfloat16, 20 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, mean, rstd, q, qs, dx, dgb)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (y, mean, rstd, q, qs, dx, dgb)))


def test_recorded_plan_replays():
    B, S, C, G = 2, 12544, 32, 4
    x, gamma, beta, dy = make(B, S, C, torch.bfloat16, 6)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    dgb = torch.empty(2, C, device="cuda")
    ws = [torch.empty(K.gn_workspace(B, S, C, G, x.dtype, b) + 4, device="cuda") for b in (False, True)]
    plan = K.LaunchPlan()

    def step():
        K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, act=3, ws=ws[0])
        K.gn_bwd(dy, x, gamma, beta, mean, rstd, dx, dgb, B, S, C, G, act=3, ws=ws[1])

    plan.record(step)
    want = [t.clone() for t in (y, mean, rstd, dx, dgb)]
    for t in (y, mean, rstd, dx, dgb):
        t.zero_()
    plan.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (y, mean, rstd, dx, dgb)))
    plan.free()


def test_a_workspace_over_an_operand_and_empty_recordings_are_refused():
    B, S, C, G = 2, 6001, 96, 12
    x, gamma, beta, dy = make(B, S, C, torch.float32, 31)
    need = K.gn_workspace(B, S, C, G, torch.float32, True)
    y, mean, rstd = torch.empty_like(x), *(torch.empty(B, G, device="cuda") for _ in range(2))
    assert y.numel() >= need > 0
    with pytest.raises(ValueError, match="ws overlaps y"):
        K.gn_fwd(x, gamma, beta, y, mean, rstd, B, S, C, G, ws=y.view(-1))
    dw, q, qs = torch.empty(64, 96, device="cuda"), *zero_codes(4096, 96)
    d = torch.zeros(4096, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ws overlaps dy"):
        K.mx8_wgrad(d, q, qs, dw, 4096, 64, 96, ws=d.view(torch.float32).view(-1))
    none = torch.empty(0, 96, device="cuda")
    plan = K.LaunchPlan()
    with pytest.raises(ValueError, match="recorded"):
        plan.record(lambda: K.gn_bwd(none, none, None, None, none, none, none, torch.empty(2, 96, device="cuda"), 0, 5,
                                     96, 12))


def zero_codes(M, C):
    return (torch.zeros(M, C, dtype=torch.uint8, device="cuda"),
            torch.full((M, K.mx8_blocks(C)), 127, dtype=torch.uint8, device="cuda"))


def test_two_streams_at_once():
    B, S, C, G = 8, 6001, 96, 12
    data = [make(B, S, C, torch.bfloat16, 30 + k) for k in range(2)]
    alone = []
    for x, gamma, beta, dy in data:
        y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, 2, True)
        alone.append((y, mean, rstd, *call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, 2, q, qs)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, (st, (x, gamma, beta, dy)) in enumerate(zip(streams, data)):
            with torch.cuda.stream(st):
                y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, 2, True)
                got[k].append((y, mean, rstd, *call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, 2, q, qs)))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(alone[k], out))


@pytest.mark.parametrize("S", [12200, 30000])
def test_one_long_image_on_four_streams(S):
    """Launches whose workgroups wait for one another share the chip: each comes out as it does alone."""
    B, C, G = 1, 128, 16
    x, gamma, beta, dy = make(B, S, C, torch.bfloat16, 50)
    y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, 2, True)
    alone = (y, mean, rstd, *call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, 2, q, qs))
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(4)] * 5:
        with torch.cuda.stream(st):
            y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, 2, True)
            got.append((y, mean, rstd, *call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, 2, q, qs)))
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(alone, out))


def test_squares_past_the_range_are_not_taken_for_zeros():
    """Values whose squares pass fp32's range have no finite variance there: rstd is 0 or NaN. Their signs
    are such that every thread's own sum is 0."""
    B, S, C, G = 1, 25600, 128, 16
    sign = 1 - 2 * (torch.arange(S, device="cuda") // 32 % 2)
    x = (1e25 * sign).to(torch.bfloat16).view(1, S, 1).expand(B, S, C).contiguous()
    one = torch.ones(C, device="cuda")
    rstd = call_fwd(x, one, one, B, S, C, G, 0, False)[2]
    assert ((rstd == 0) | rstd.isnan()).all()


def test_offsets_past_32_bits():
    """2.15e9 values (4.3 GB): the last image comes out as it does alone."""
    B, S, C, G = 5, 419431, 1024, 128
    assert B * S * C > 1 << 31
    x = torch.empty(B, S, C, dtype=torch.bfloat16, device="cuda")
    dy = torch.empty_like(x)
    for b in range(B):
        x[b].normal_(0.1 * b, 1)
        dy[b].normal_()
    g = torch.Generator(device="cuda").manual_seed(1)
    gamma, beta = (torch.randn(C, generator=g, device="cuda") for _ in range(2))
    y, mean, rstd, q, qs = call_fwd(x, gamma, beta, B, S, C, G, 1, True)
    y1, mean1, rstd1, q1, qs1 = call_fwd(x[-1:].clone(), gamma, beta, 1, S, C, G, 1, True)
    O.within(mean[-1:], mean1.double(), 1e-5 * torch.ones_like(mean1).double())
    assert torch.equal(q[-S:], q1) and torch.equal(qs[-S:], qs1)
    assert (y[-1].float() - y1[0].float()).abs().max() <= 2 * 2.0 ** -8 * y1.float().abs().max()
    del y, y1, q1, qs1
    dx, _ = call_bwd(dy, None, gamma, beta, mean, rstd, B, S, C, G, 1, q, qs)
    dx1, _ = call_bwd(dy[-1:].clone(), None, gamma, beta, mean[-1:].clone(), rstd[-1:].clone(), 1, S, C, G, 1,
                      q[-S:].clone(), qs[-S:].clone())
    assert (dx[-1].float() - dx1[0].float()).abs().max() <= 2 * 2.0 ** -8 * dx1.float().abs().max()
