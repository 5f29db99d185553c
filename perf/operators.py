"""Measured cases of the group-norm and 8-bit activation-checkpoint operators (pgdist.ops.kernels).

Five operators, as a training step of a channels-last network with group norm calls them:

  gn_fwd   y = act(group_norm(x) * gamma + beta), and the 8-bit checkpoint of x in the same pass
  gn_bwd   dx, dgamma, dbeta from dy and x, or from dy and the 8-bit checkpoint of x
  pack     [M, C] values -> e4m3 codes and one power-of-two scale for every 32 channels of a row
  unpack   the values that codes and scales stand for
  wgrad    dW = dY^T X and db of a linear layer or 1x1 convolution whose input was kept in 8 bits

``run`` computes them with elementary torch operations, or (``own``) through the framework's entry
points; ``exact`` computes them from their definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("none", "relu", "relu6", "silu")
EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # the last feature map of one image: a request served on its own, all latency
        dict(name="gn_fwd_one_image", op="gn_fwd", B=1, S=49, C=1280, G=160, act="relu6", dtype="bf16", ck=False),
        # an expand layer at 56 x 56 in training: the checkpoint of x leaves in the same pass
        dict(name="gn_fwd_train_ck", op="gn_fwd", B=128, S=3136, C=144, G=18, act="relu6", dtype="bf16", ck=True),
        # full precision, sizes that no tile divides
        dict(name="gn_fwd_f32_ragged", op="gn_fwd", B=7, S=3249, C=100, G=10, act="silu", dtype="fp32", ck=False),
        # a mid-network layer of a 96-image batch, backward from the checkpoint
        dict(name="gn_bwd_ck", op="gn_bwd", B=96, S=784, C=192, G=24, act="relu6", dtype="bf16", ck=True),
        # the widest map of a 128-image batch, backward from x itself: the largest
        dict(name="gn_bwd_large", op="gn_bwd", B=128, S=12544, C=96, G=12, act="relu6", dtype="bf16", ck=False),
        # a small map of a small batch
        dict(name="pack_small", op="pack", M=1568, C=576, dtype="bf16"),
        # the expand layer above, packed on its own
        dict(name="pack_large", op="pack", M=401408, C=144, dtype="bf16"),
        # odd rows and channels, half precision
        dict(name="unpack_ragged", op="unpack", M=24999, C=75, dtype="fp16"),
        # a mid-network layer
        dict(name="unpack_large", op="unpack", M=100352, C=960, dtype="bf16"),
        # the classifier of a 128-image batch: few rows
        dict(name="wgrad_classifier", op="wgrad", M=128, N=1000, K=2048, dtype="bf16"),
        # an expand convolution at 56 x 56: many rows, a small weight, bound by what it reads
        dict(name="wgrad_narrow", op="wgrad", M=401408, N=144, K=24, dtype="bf16"),
        # a wide layer: bound by the matrix cores
        dict(name="wgrad_wide", op="wgrad", M=25088, N=1024, K=1024, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dtype(rng, wide=True):
    return rng.choice(("bf16", "bf16", "fp16", "fp32") if wide else ("bf16", "bf16", "fp16"))


def draw(rng):
    op = rng.choice(("gn_fwd", "gn_bwd", "pack", "unpack", "wgrad"))
    if op in ("gn_fwd", "gn_bwd"):
        # channels: eights as the models have them, or any number of groups of any width
        if rng.random() < 0.6:
            cg, G = 8, _log(rng, 1, 160)
        else:
            cg, G = _log(rng, 1, 48), _log(rng, 1, 40)
        dtype = _dtype(rng)
        most = 40_000_000 if dtype == "fp32" else 100_000_000   # values: no more than the largest listed case
        B = _log(rng, 1, 128)
        S = _log(rng, 1, 12544)
        S = max(-(-64 // cg), min(S, most // (B * cg * G)))     # statistics of 64 values at least
        return dict(op=op, B=B, S=S, C=cg * G, G=G, act=rng.choice(ACTS), dtype=dtype, ck=rng.random() < 0.5)
    if op in ("pack", "unpack"):
        C = 8 * _log(rng, 1, 256) if rng.random() < 0.6 else _log(rng, 1, 2048)
        return dict(op=op, M=max(1, min(_log(rng, 1, 400_000), 60_000_000 // C)), C=C, dtype=_dtype(rng))
    N, K = (8 * _log(rng, 1, 160) if rng.random() < 0.6 else _log(rng, 1, 1280) for _ in range(2))
    M = max(1, min(_log(rng, 1, 400_000), 20_000_000_000 // (N * K), 80_000_000 // (N + K)))
    return dict(op=op, M=M, N=N, K=K, dtype=_dtype(rng, wide=False))


# --------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _activations(gen, B, S, C, dt):
    """A convolution's output: every channel has its own mean and spread, every image its own level."""
    x = _randn(gen, B, S, C)
    x.mul_(0.5 + _rand(gen, C)).add_(0.7 * _randn(gen, C)).add_(0.3 * _randn(gen, B, 1, 1))
    return x.to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)

    def empty(*shape, dtype=dt):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    def codes(M, C):
        return empty(M, C, dtype=torch.uint8), empty(M, -(-C // BLOCK), dtype=torch.uint8)

    op = case["op"]
    if op in ("gn_fwd", "gn_bwd"):
        B, S, C, G = case["B"], case["S"], case["C"], case["G"]
        s["x"] = _activations(gen, B, S, C, dt)
        s["gamma"] = 1 + 0.2 * _randn(gen, C)
        s["beta"] = 0.3 * _randn(gen, C)
        if op == "gn_fwd":
            s["y"] = empty(B, S, C)
            s["mean"], s["rstd"] = empty(B, G, dtype=torch.float32), empty(B, G, dtype=torch.float32)
            s["q"], s["qs"] = codes(B * S, C) if case["ck"] else (None, None)
        else:   # what the forward pass left: the statistics, and x or its checkpoint
            var, mean = torch.var_mean(s["x"].view(B, S, G, C // G).double(), dim=(1, 3), unbiased=False)
            s["mean"], s["rstd"] = mean.float(), (var + EPS).rsqrt().float()
            s["dy"] = (_randn(gen, B, S, C) * torch.exp(_randn(gen, B, 1, 1))).to(dt)
            s["q"], s["qs"] = _pack(s["x"].view(B * S, C)) if case["ck"] else (None, None)
            if case["ck"]:
                s["x"] = None
            s["dx"], s["dgb"] = empty(B, S, C), empty(2, C, dtype=torch.float32)
    elif op == "pack":
        s["x"] = _activations(gen, 1, case["M"], case["C"], dt).view(case["M"], case["C"])
        s["q"], s["qs"] = codes(case["M"], case["C"])
    elif op == "unpack":
        s["q"], s["qs"] = _pack(_activations(gen, 1, case["M"], case["C"], dt).view(case["M"], case["C"]))
        s["x"] = empty(case["M"], case["C"])
    else:
        M, N, K = case["M"], case["N"], case["K"]
        s["dy"] = _randn(gen, M, N).to(dt)
        s["q"], s["qs"] = _pack(_activations(gen, 1, M, K, dt).view(M, K))
        s["dw"], s["db"] = empty(N, K, dtype=torch.float32), empty(N, dtype=torch.float32)
    return s


# --------------------------------------------------------------------------- the plain forms
def _pow2(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(x):
    """codes (uint8) and scales (uint8: exponent + 127) of [M, C] values."""
    M, C = x.shape
    nb = -(-C // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - C)).view(M, nb, BLOCK)
    frac, ex = torch.frexp(v.abs().amax(2))               # amax = frac * 2^ex; 448 = 0.875 * 2^9
    e = (ex - 9 + (frac > 0.875).to(ex.dtype)).clamp(-117, 120)
    e = torch.where(frac == 0, -117, e)
    q = (v * _pow2(-e).unsqueeze(2)).to(torch.float8_e4m3fn).view(M, nb * BLOCK)[:, :C]
    return q.contiguous().view(torch.uint8), (e + 127).to(torch.uint8)


def _unpack(q, qs):
    """the fp32 values that codes and scales stand for."""
    scale = _pow2(qs.to(torch.int32) - 127).repeat_interleave(BLOCK, dim=1)[:, :q.shape[1]]
    return q.view(torch.float8_e4m3fn).float() * scale


def _values(q, qs):
    return q.view(torch.float8_e4m3fn), qs.view(torch.float8_e8m0fnu)


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "relu6":
        return z.clamp(0, 6)
    return z * torch.sigmoid(z) if act == "silu" else z


def _plain_gn_fwd(s, B, S, C, G, act, ck):
    x = s["x"].float().view(B, S, G, C // G)
    mean = x.mean(dim=(1, 3))
    d = x - mean.view(B, 1, G, 1)
    rstd = (d.square().mean(dim=(1, 3)) + EPS).rsqrt()
    z = (d * rstd.view(B, 1, G, 1)).view(B, S, C) * s["gamma"] + s["beta"]
    out = [_act(z, act).to(s["x"].dtype), mean, rstd]
    return out + list(_values(*_pack(s["x"].view(B * S, C)))) if ck else out


def _plain_gn_bwd(s, B, S, C, G, act, ck):
    x = _unpack(s["q"], s["qs"]) if ck else s["x"].float()
    mean, rstd = s["mean"].view(B, 1, G, 1), s["rstd"].view(B, 1, G, 1)
    xh = ((x.view(B, S, G, C // G) - mean) * rstd).view(B, S, C)
    dz = s["dy"].float()
    if act == "silu":
        z = xh * s["gamma"] + s["beta"]
        sig = torch.sigmoid(z)
        dz = dz * (sig * (1 + z * (1 - sig)))
    elif act != "none":   # which side of the border z lies on is decided in 64 bits
        z = ((x.double().view(B, S, G, C // G) - mean) * rstd.double()).view(B, S, C) * s["gamma"].double() + s["beta"]
        dz = torch.where((z > 0) & (z < 6) if act == "relu6" else z > 0, dz, 0.0)
    dgamma, dbeta = (dz * xh).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    t, xg = (dz * s["gamma"]).view(B, S, G, C // G), xh.view(B, S, G, C // G)
    m1, m2 = t.mean(dim=(1, 3), keepdim=True), (t * xg).mean(dim=(1, 3), keepdim=True)
    dx = rstd * (t - m1 - xg * m2)
    return [dx.view(B, S, C).to(s["dy"].dtype), dgamma, dbeta]


_K = None


def _kernels():
    """The framework's entry points, imported when they are first asked for."""
    global _K
    if _K is None:
        import pgdist  # noqa: F401
        from pgdist.ops import kernels
        _K = kernels
    return _K


def run(s):
    c = s["case"]
    op = c["op"]
    K = _kernels() if own else None
    if op in ("gn_fwd", "gn_bwd"):
        B, S, C, G = c["B"], c["S"], c["C"], c["G"]
        if not own:
            return (_plain_gn_fwd if op == "gn_fwd" else _plain_gn_bwd)(s, B, S, C, G, c["act"], c["ck"])
        act = (K.GN_NONE, K.GN_RELU, K.GN_RELU6, K.GN_SILU)[ACTS.index(c["act"])]
        if op == "gn_fwd":
            K.gn_fwd(s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"], B, S, C, G, eps=EPS, act=act,
                     q=s["q"], qs=s["qs"])
            out = [s["y"], s["mean"], s["rstd"]]
            return out + list(_values(s["q"], s["qs"])) if c["ck"] else out
        K.gn_bwd(s["dy"], s["x"], s["gamma"], s["beta"], s["mean"], s["rstd"], s["dx"], s["dgb"], B, S, C, G, act=act,
                 q=s["q"], qs=s["qs"])
        return [s["dx"], s["dgb"][0], s["dgb"][1]]
    if op == "pack":
        if not own:
            return list(_values(*_pack(s["x"])))
        K.mx8_pack(s["x"], s["q"], s["qs"], c["M"], c["C"])
        return list(_values(s["q"], s["qs"]))
    if op == "unpack":
        if not own:
            v = _unpack(s["q"], s["qs"])   # half precision ends at 65504: what rounds up past that stays finite
            return (v.clamp(-65504, 65504) if c["dtype"] == "fp16" else v).to(s["x"].dtype)
        K.mx8_unpack(s["q"], s["qs"], s["x"], c["M"], c["C"])
        return s["x"]
    if not own:
        dy = s["dy"].float()
        return [dy.t() @ _unpack(s["q"], s["qs"]), dy.sum(0)]
    K.mx8_wgrad(s["dy"], s["q"], s["qs"], s["dw"], c["M"], c["N"], c["K"], db=s["db"])
    return [s["dw"], s["db"]]


# --------------------------------------------------------------------------- work and definitions
def work(case):
    op = case["op"]
    if op in ("gn_fwd", "gn_bwd"):
        n, e = case["B"] * case["S"] * case["C"], DTYPES[case["dtype"]].itemsize
        q = case["B"] * case["S"] * (case["C"] + -(-case["C"] // BLOCK))
        small = 8 * case["C"] + 8 * case["B"] * case["G"]
        if op == "gn_fwd":
            return {"bytes": 2 * n * e + (q if case["ck"] else 0) + small, "flops": 8 * n}
        return {"bytes": 2 * n * e + (q if case["ck"] else n * e) + small + 8 * case["C"], "flops": 16 * n}
    if op in ("pack", "unpack"):
        M, C = case["M"], case["C"]
        return {"bytes": M * (C * DTYPES[case["dtype"]].itemsize + C + -(-C // BLOCK)), "flops": 2 * M * C}
    M, N, K_ = case["M"], case["N"], case["K"]
    return {"bytes": M * (N * DTYPES[case["dtype"]].itemsize + K_ + -(-K_ // BLOCK)) + 4 * N * (K_ + 1),
            "flops": 2 * M * N * K_ + M * N}


def _grid():
    """The 127 values of e4m3 from 0 to 448, in code order."""
    c = torch.arange(127, device="cuda")
    ex, man = (c >> 3).double(), (c & 7).double()
    return torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * torch.exp2(ex - 7))


def _exact_pack(x):
    M, C = x.shape
    nb = -(-C // BLOCK)
    v = torch.zeros(M, nb * BLOCK, dtype=torch.float64, device="cuda")
    v[:, :C] = x.double()
    v = v.view(M, nb, BLOCK)
    top = v.abs().amax(2)
    ex = torch.ceil(torch.log2(top / 448)).clamp(-117, 120)   # log2(0) clamps to -117
    ex = torch.where(top > 448 * torch.exp2(ex), ex + 1, ex)
    ex = torch.where((top <= 448 * torch.exp2(ex - 1)) & (ex > -117), ex - 1, ex)
    scale = torch.exp2(ex)
    u = v / scale.unsqueeze(2)
    g = _grid()
    mid = (g[1:] + g[:-1]) / 2
    a = u.abs()
    lo = torch.bucketize(a, mid)                # first code whose upper midpoint is >= a
    tie = a == mid[lo.clamp(max=125)]           # half way between lo and lo + 1: the even one
    code = lo + (tie & (lo < 126) & (lo % 2 == 1)).long()
    return (g[code] * torch.sign(u)).view(M, nb * BLOCK)[:, :C], scale


def _exact_unpack(q, qs):
    g = torch.cat([_grid(), torch.full((1,), float("nan"), dtype=torch.float64, device="cuda")])
    v = g[(q & 127).long()] * (1 - 2 * (q >> 7).double())
    return v * torch.exp2(qs.double() - 127).repeat_interleave(BLOCK, dim=1)[:, :q.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "pack":
        return list(_exact_pack(s["x"]))
    if op == "unpack":
        v = _exact_unpack(s["q"], s["qs"])
        return v.clamp(-65504.0, 65504.0) if case["dtype"] == "fp16" else v
    if op == "wgrad":
        dy = s["dy"].double()
        return [torch.mm(dy.t().contiguous(), _exact_unpack(s["q"], s["qs"])), dy.sum(0)]
    B, S, C, G, act = case["B"], case["S"], case["C"], case["G"], case["act"]
    gamma, beta = s["gamma"].double().view(G, C // G), s["beta"].double().view(G, C // G)
    if op == "gn_fwd":
        v = s["x"].double().view(B, S, G, C // G)
        mean = v.sum(dim=(1, 3)) / (S * (C // G))
        v = v - mean[:, None, :, None]
        rstd = 1 / torch.sqrt((v * v).sum(dim=(1, 3)) / (S * (C // G)) + EPS)
        v = v * rstd[:, None, :, None] * gamma + beta
        if act in ("relu", "relu6"):
            v = torch.where(v < 0, 0.0, v)
        if act == "relu6":
            v = torch.where(v > 6, 6.0, v)
        if act == "silu":
            v = v / (1 + torch.exp(-v))
        out = [v.view(B, S, C), mean, rstd]
        return out + list(_exact_pack(s["x"].view(B * S, C))) if case["ck"] else out
    x = _exact_unpack(s["q"], s["qs"]) if case["ck"] else s["x"].double()
    rstd = s["rstd"].double()[:, None, :, None]
    xh = (x.view(B, S, G, C // G) - s["mean"].double()[:, None, :, None]) * rstd
    z = xh * gamma + beta
    g = s["dy"].double().view(B, S, G, C // G)
    if act == "silu":   # d/dz z/(1+e^-z) = (1 + e^-z (1 + z)) / (1 + e^-z)^2
        w = torch.exp(-z)
        g = g * (1 + w * (1 + z)) / (1 + w) ** 2
    elif act == "relu":
        g = g * (z > 0)
    elif act == "relu6":
        g = g * ((z > 0) & (z < 6))
    dgamma, dbeta = (g * xh).sum(dim=(0, 1)).view(C), g.sum(dim=(0, 1)).view(C)
    g = g * gamma
    m = S * (C // G)
    dx = rstd * (g - g.sum(dim=(1, 3), keepdim=True) / m - xh * ((g * xh).sum(dim=(1, 3), keepdim=True) / m))
    return [dx.view(B, S, C), dgamma, dbeta]
