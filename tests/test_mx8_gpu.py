"""8-bit activation checkpoints: pack, unpack, and the weight gradient read from one."""
import pytest
import torch

import gn_oracle as O
from pgdist.ops import kernels as K

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def pack(x):
    M, C = x.shape
    q = torch.full((M, C), 255, dtype=torch.uint8, device="cuda")
    qs = torch.full((M, K.mx8_blocks(C)), 255, dtype=torch.uint8, device="cuda")
    K.mx8_pack(x, q, qs, M, C)
    return q, qs


def values(M, C, dt, seed=0):
    """Rows of every magnitude the type holds, and ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, C, generator=g, device="cuda")
    lim = 12 if dt == torch.float16 else 100
    e = torch.randint(-lim, lim + 1, (M, 1), generator=g, device="cuda").float()
    x = torch.where(torch.arange(M, device="cuda").view(M, 1) % 2 == 0, x, x * torch.exp2(e))
    return x.to(dt)


SHAPES = [(1, 1), (1, 31), (1, 32), (1, 33), (7, 8), (5, 24), (3, 100), (64, 144), (33, 75), (1568, 576), (2000, 16),
          (9, 2049), (257, 960), (1, 40000), (4099, 2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack(shape, dtype):
    x = values(*shape, DT[dtype], shape[0])
    q, qs = pack(x)
    wq, ws = O.pack(x)
    assert torch.equal(qs, ws) and torch.equal(q, wq)
    want = O.unpack(q, qs)
    # a normal code is half a step of e4m3 off at most, 2^-4 of the value; a subnormal one 2^-10 of its scale
    step = torch.exp2(qs.double() - 127).repeat_interleave(32, 1)[:, :shape[1]]
    assert ((want - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * step)).all()
    for dt in DT.values():
        out = torch.empty(shape, dtype=dt, device="cuda")
        K.mx8_unpack(q, qs, out, *shape)
        w = want.clamp(-65504, 65504) if dt == torch.float16 else want
        assert torch.equal(out, w.to(dt))
        if dt != torch.float16:
            assert torch.equal(out.double(), want)   # exact


def test_special_values():
    rows = [[0.0] * 4, [-0.0, 0.0, 1.0, -1.0], [float("nan"), 1.0, 2.0, 448.0], [float("inf"), -float("inf"), 3.0, 0.5],
            [float("nan")] * 4, [448.0, 447.0, 1.0, 1e-3], [449.0, 448.0, 464.0, 1.0], [3.4e38, -3.4e38, 1.0, 0.0],
            [1e-38, 1e-39, -1e-45, 0.0], [2.0 ** -126, 2.0 ** -125, 2.0 ** -117, 2.0 ** -120],
            [65504.0, 1.0, -65504.0, 2.0], [1.0625, 1.1875, 448.0, 25.0], [2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 448.0]]
    x = torch.tensor(rows, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        q, qs = pack(x.to(dt))
        wq, ws = O.pack(x.to(dt))
        assert torch.equal(qs, ws)
        assert torch.equal(torch.where((wq & 127) == 127, q & 127, q), wq)
        out = torch.empty_like(x)
        K.mx8_unpack(q, qs, out, *x.shape)
        assert torch.equal(torch.isnan(out), ~torch.isfinite(x.to(dt)))


def test_every_code_of_every_scale_decodes_exactly():
    q = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(238, 1)
    qs = torch.arange(10, 248, dtype=torch.uint8, device="cuda").view(238, 1).repeat(1, 8)
    want = O.unpack(q, qs)
    for dt in DT.values():
        out = torch.empty(q.shape, dtype=dt, device="cuda")
        K.mx8_unpack(q, qs, out, *q.shape)
        w = want.clamp(-65504, 65504) if dt == torch.float16 else want
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(out), nan)
        # 2^128 and above is past fp32's end: the largest codes of the largest scale only
        assert torch.equal(out[~nan], w.to(dt)[~nan])


def wgrad_case(M, N, Kd, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(M, N, generator=g, device="cuda").to(dt)
    x = (torch.randn(M, Kd, generator=g, device="cuda") * torch.exp2(torch.randint(-3, 4, (M, 1), generator=g,
                                                                                  device="cuda").float())).to(dt)
    return dy, *O.pack(x)


WG = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (31, 16, 33), (128, 1000, 2048), (100, 10, 1280), (200, 144, 24), (777, 24, 144),
      (513, 65, 129), (64, 256, 256), (2000, 96, 576), (20000, 17, 19), (9000, 320, 40), (33, 300, 257), (4097, 128, 128)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 12, 15, 17, 31, 33, 34, 36, 39, 41, 63, 65, 95, 97, 129, 1001])
def test_every_row_length_and_nothing_behind(C, dtype):
    """Rows that begin at any alignment, matrices that end inside a vector, and the bytes behind them."""
    for M in (1, 2, 5, 700):
        g = torch.Generator(device="cuda").manual_seed(C * M)
        x = (torch.randn(M, C, generator=g, device="cuda") * 2.0 ** torch.randint(-9, 9, (M, 1), generator=g, device="cuda")).to(DT[dtype])
        q = torch.full((M * C + 64,), 77, dtype=torch.uint8, device="cuda")
        qs = torch.full((M * K.mx8_blocks(C) + 64,), 77, dtype=torch.uint8, device="cuda")
        K.mx8_pack(x, q[:M * C].view(M, C), qs[:-64].view(M, -1), M, C)
        wq, ws = O.pack(x)
        assert torch.equal(q[:M * C].view(M, C), wq) and torch.equal(qs[:-64].view(M, -1), ws)
        y = torch.full((M * C + 64,), 77.0, dtype=DT[dtype], device="cuda")
        K.mx8_unpack(wq, ws, y[:M * C].view(M, C), M, C)
        assert torch.equal(y[:M * C].view(M, C), O.unpack(wq, ws).to(DT[dtype]))
        assert (q[M * C:] == 77).all() and (qs[-64:] == 77).all() and (y[M * C:] == 77).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mnk", [(1, 1, 1), (3, 5, 7), (129, 33, 31), (1025, 65, 127), (641, 257, 3), (30001, 129, 65)])
def test_wgrad_takes_nothing_from_behind_its_operands(mnk, dtype):
    """Rows of odd lengths end inside a word: NaN in its other half, and after it, stays outside."""
    M, N, Kd = mnk
    dy, q, qs = wgrad_case(M, N, Kd, DT[dtype], M + 1)

    def inside(t, fill):
        big = torch.full((t.numel() + 4096,), fill, dtype=t.dtype, device="cuda")
        big[:t.numel()] = t.reshape(-1)
        return big[:t.numel()].view(t.shape)

    out = []
    for d, c, e in ((dy, q, qs), (inside(dy, float("nan")), inside(q, 127), inside(qs, 254))):
        dw, db = torch.full((N, Kd), float("nan"), device="cuda"), torch.full((N,), float("nan"), device="cuda")
        K.mx8_wgrad(d, c, e, dw, M, N, Kd, db=db)
        out.append((dw, db))
    assert torch.isfinite(out[0][0]).all() and torch.isfinite(out[0][1]).all()
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mnk", WG)
def test_wgrad(mnk, dtype):
    M, N, Kd = mnk
    dy, q, qs = wgrad_case(M, N, Kd, DT[dtype], M)
    dw = torch.full((N, Kd), float("nan"), device="cuda")
    db = torch.full((N,), float("nan"), device="cuda")
    K.mx8_wgrad(dy, q, qs, dw, M, N, Kd, db=db)
    x = O.unpack(q, qs)
    d = dy.double()
    want, mag = d.t().contiguous() @ x, d.abs().t().contiguous() @ x.abs()
    # every product is exact in fp32 (12 significant bits); at most M + 64 additions, each u off
    O.within(dw, want, (M + 64) * O.U * mag)
    O.within(db, O.sums(d), (M + 64) * O.U * O.sums(d.abs()))
    # roundings are as often up as down: over the matrix they add as a random walk, u sqrt(M / 6) of the norm
    assert (dw.double() - want).norm() <= 4 * O.U * (M + 1) ** 0.5 * want.norm() + 1e-30
    again = torch.empty_like(dw)
    K.mx8_wgrad(dy, q, qs, again, M, N, Kd)
    assert torch.equal(again, dw)


def test_wgrad_special_values():
    """A NaN in row m, column n of dY reaches row n of dW alone; one in X, column k alone."""
    M, N, Kd = 100, 40, 70
    dy, q, qs = wgrad_case(M, N, Kd, torch.bfloat16, 1)
    clean = torch.empty(N, Kd, device="cuda")
    K.mx8_wgrad(dy, q, qs, clean, M, N, Kd)
    dy[17, 3] = float("nan")
    q[55, 60] = 127
    dw, db = torch.empty(N, Kd, device="cuda"), torch.empty(N, device="cuda")
    K.mx8_wgrad(dy, q, qs, dw, M, N, Kd, db=db)
    hit = torch.zeros(N, Kd, dtype=torch.bool, device="cuda")
    hit[3] = True
    hit[:, 60] = True
    assert torch.isnan(dw[hit]).all() and torch.equal(dw[~hit], clean[~hit])
    assert torch.isnan(db[3]) and torch.isfinite(db[:3]).all() and torch.isfinite(db[4:]).all()


def test_wgrad_far_half_precision_values_stay_finite():
    x = torch.full((64, 32), 65504.0, dtype=torch.float16, device="cuda")
    q, qs = O.pack(x)
    dy = torch.ones(64, 8, dtype=torch.float16, device="cuda")
    dw = torch.empty(8, 32, device="cuda")
    K.mx8_wgrad(dy, q, qs, dw, 64, 8, 32)
    assert (dw == 64 * 65504.0).all()


def test_empty_sizes():
    dw, db = torch.ones(4, 40, device="cuda"), torch.ones(4, device="cuda")
    dy = torch.empty(0, 4, dtype=torch.bfloat16, device="cuda")
    q, qs = pack(torch.empty(0, 40, dtype=torch.bfloat16, device="cuda"))
    K.mx8_wgrad(dy, q, qs, dw, 0, 4, 40, db=db)
    assert (dw == 0).all() and (db == 0).all()
    K.mx8_unpack(q, qs, torch.empty(0, 40, device="cuda"), 0, 40)


def test_nothing_written_behind():
    for M, C in ((33, 75), (100, 144), (7, 32)):
        x = values(M, C, torch.bfloat16, 2)
        n, ns = M * C, M * K.mx8_blocks(C)
        q, qs = torch.full((n + 64,), 9, dtype=torch.uint8, device="cuda"), torch.full((ns + 64,), 9, dtype=torch.uint8, device="cuda")
        K.mx8_pack(x, q[:n], qs[:ns], M, C)
        out = torch.full((n + 64,), 3.0, dtype=torch.bfloat16, device="cuda")
        K.mx8_unpack(q[:n], qs[:ns], out[:n], M, C)
        dw, db = torch.full((C * C + 64,), 3.0, device="cuda"), torch.full((C + 64,), 3.0, device="cuda")
        K.mx8_wgrad(x, q[:n], qs[:ns], dw[:C * C], M, C, C, db=db[:C])
        assert (q[n:] == 9).all() and (qs[ns:] == 9).all() and (out[n:] == 3).all()
        assert (dw[C * C:] == 3).all() and (db[C:] == 3).all()


def test_captured_and_replayed():
    M, N, Kd = 5000, 96, 200
    x = values(M, Kd, torch.bfloat16, 3)
    dy, _, _ = wgrad_case(M, N, Kd, torch.bfloat16, 3)
    q, qs = torch.empty(M, Kd, dtype=torch.uint8, device="cuda"), torch.empty(M, K.mx8_blocks(Kd), dtype=torch.uint8, device="cuda")
    out, dw, db = torch.empty_like(x), torch.empty(N, Kd, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.empty(K.mx8_wgrad_workspace(M, N, Kd) + 4, device="cuda")

    def step():
        K.mx8_pack(x, q, qs, M, Kd)
        K.mx8_unpack(q, qs, out, M, Kd)
        K.mx8_wgrad(dy, q, qs, dw, M, N, Kd, db=db, ws=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, qs, out, dw, db)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (q, qs, out, dw, db)))


def test_two_streams_at_once():
    M, N, Kd = 30000, 144, 96
    data = [wgrad_case(M, N, Kd, torch.bfloat16, k) for k in range(2)]
    want = []
    for dy, q, qs in data:
        want.append((torch.empty(N, Kd, device="cuda"), torch.empty(N, device="cuda")))
        K.mx8_wgrad(dy, q, qs, want[-1][0], M, N, Kd, db=want[-1][1])
    torch.cuda.synchronize()
    got = [[], []]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                o = (torch.empty(N, Kd, device="cuda"), torch.empty(N, device="cuda"))
                K.mx8_wgrad(*data[k], o[0], M, N, Kd, db=o[1])
                got[k].append(o)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for o in got[k] for a, b in zip(o, want[k]))


def test_offsets_past_32_bits():
    M, C = (1 << 31) // 1000 + 7, 1000
    x = torch.empty(M, C, dtype=torch.bfloat16, device="cuda").normal_()
    q, qs = pack(x)
    wq, ws = O.pack(x[-1000:])
    assert torch.equal(q[-1000:], wq) and torch.equal(qs[-1000:], ws)
    out = torch.empty_like(x)
    K.mx8_unpack(q, qs, out, M, C)
    assert torch.equal(out[-1000:].double(), O.unpack(q[-1000:], qs[-1000:]))
    del out
    # only the rows behind the 2^31st value of dY count
    N = 1000
    cut = 1500
    x[:-cut] = 0
    dw = torch.empty(N, C, device="cuda")
    K.mx8_wgrad(x, q, qs, dw, M, N, C)
    d, v = x[-cut:].double(), O.unpack(q[-cut:], qs[-cut:])
    want, mag = d.t().contiguous() @ v, d.abs().t().contiguous() @ v.abs()
    O.within(dw, want, (cut + 64) * O.U * mag)
