"""64-bit oracles of the group-norm and 8-bit checkpoint operators, and the error bounds their tests use.

Rounding counts: u = 2^-24 is half a step of fp32, half(t) half a step of the output type.  A sum of n
values of which any thread adds at most L in a row, followed by a tree, is off by at most
(L + 32) u times the sum of magnitudes."""
import torch

U = 2.0 ** -24


def half(dt):
    return torch.finfo(dt).eps / 2


def grid(device="cpu"):
    """The 127 values of e4m3 from 0 to 448, in code order."""
    c = torch.arange(127, device=device)
    ex, man = (c >> 3).double(), (c & 7).double()
    return torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * torch.exp2(ex - 7))


def pack(x):
    """(codes, exponent bytes) of [M, C] by search over the value grid."""
    M, C = x.shape
    nb = -(-C // 32)
    v = torch.zeros(M, nb * 32, dtype=torch.float64, device=x.device)
    v[:, :C] = x.double()
    v = v.view(M, nb, 32)
    fin = torch.isfinite(v)
    top = torch.where(fin, v.abs(), 0.0).amax(2)
    e = torch.full_like(top, -117)
    for k in range(-116, 121):          # the least exponent that holds the block
        e = torch.where(top > 448 * 2.0 ** (k - 1), float(k), e)
    u = torch.where(fin, v, 0.0) / torch.exp2(e).unsqueeze(2)
    g = grid(x.device)
    mid = (g[1:] + g[:-1]) / 2
    a = u.abs()
    lo = torch.bucketize(a, mid)
    tie = a == mid[lo.clamp(max=125)]
    code = lo + (tie & (lo < 126) & (lo % 2 == 1)).long()
    code = torch.where(fin, code + 128 * torch.signbit(u).long(), 127)
    return code.view(M, nb * 32)[:, :C].to(torch.uint8).contiguous(), (e + 127).to(torch.uint8)


def unpack(q, qs):
    g = torch.cat([grid(q.device), torch.full((1,), float("nan"), dtype=torch.float64, device=q.device)])
    v = g[(q & 127).long()] * (1 - 2 * (q >> 7).double())
    return v * torch.exp2(qs.double() - 127).repeat_interleave(32, dim=1)[:, :q.shape[1]]


def act(z, a):
    if a == 1:
        return torch.where(z < 0, 0.0, z)
    if a == 2:
        return torch.where(z < 0, 0.0, torch.where(z > 6, 6.0, z))
    return z * torch.sigmoid(z) if a == 3 else z


def dact(z, a):
    if a == 1:
        return (z > 0).double()
    if a == 2:
        return ((z > 0) & (z < 6)).double()
    if a == 3:
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def sums(v):
    """Sum over dim 0, 256 values at a time. torch's own sum of many values to few results works across
    workgroups, and one in some 1500 such sums (1200004 doubles to 3) came out a hundredth off."""
    while v.shape[0] > 256:
        n = -(-v.shape[0] // 256)
        w = torch.zeros(n * 256, *v.shape[1:], dtype=v.dtype, device=v.device)
        w[:v.shape[0]] = v
        v = w.view(n, 256, *v.shape[1:]).sum(1)
    return v.sum(0)


def _means(v):
    """[B, S, G, cg] -> [B, G]"""
    return sums(v.transpose(0, 1)).sum(2) / (v.shape[1] * v.shape[3])


def _rep(t, B, S, C, G):
    return t.double().view(B, 1, G, 1).expand(B, S, G, C // G).reshape(B, S, C)


def fwd(x, gamma, beta, B, S, C, G, eps, a):
    """y, mean, rstd in 64 bits and bounds on y, mean, rstd."""
    v = x.double().view(B, S, G, C // G)
    n = S * (C // G)
    mean = _means(v)
    var = _means((v - mean.view(B, 1, G, 1)).square())
    rstd = 1 / torch.sqrt(var + eps)
    g = torch.ones(C, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    d = x.double().view(B, S, C) - _rep(mean, B, S, C, G)
    rs = _rep(rstd, B, S, C, G)
    z = d * rs * g + b
    t = (n / 64 + 32) * U
    em = t * _means(v.abs()) + U * mean.abs()
    # the squares' sum is off by t of itself, and by the mean's error squared
    er = rstd * (t + 8 * U) + 0.5 * rstd ** 3 * em ** 2
    y = act(z, a)
    ez = g.abs() * (rs * _rep(em, B, S, C, G) + d.abs() * _rep(er, B, S, C, G)) + 6 * U * ((d * rs * g).abs() + b.abs() + z.abs())
    if a == 3:
        ez = 1.1 * ez + 2.0 ** -20 * z.abs() * (1 + z.abs()) * torch.sigmoid(z)
    return (y, mean, rstd), (ez + half(x.dtype) * y.abs() + tiny(x.dtype), em, er)


def tiny(dt):
    """half a step of the smallest (subnormal) values of an output type"""
    return {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}.get(dt, 0.0)


def bwd(dy, x, gamma, beta, mean, rstd, B, S, C, G, a):
    """dx, dgamma, dbeta in 64 bits (x: the values that stand for the input) and their bounds."""
    dt = dy.dtype
    dev = dy.device
    g = torch.ones(C, dtype=torch.float64, device=dev) if gamma is None else gamma.double()
    b = torch.zeros(C, dtype=torch.float64, device=dev) if beta is None else beta.double()
    rs = _rep(rstd, B, S, C, G)
    xh = (x.double().view(B, S, C) - _rep(mean, B, S, C, G)) * rs
    z = xh * g + b
    dyd = dy.double().view(B, S, C)
    dz = dyd * dact(z, a)
    n = S * (C // G)

    def gmean(t):
        return _rep(_means(t.view(B, S, G, C // G)), B, S, C, G)

    m1, m2 = gmean(dz * g), gmean(dz * g * xh)
    dx = rs * (dz * g - m1 - xh * m2)
    edz = 4 * U * dz.abs()
    if a == 3:   # sigmoid and its slope carry the exponential's error, larger where |z| is
        edz = edz + 2.0 ** -19 * dyd.abs() * (1 + z.abs()) * torch.sigmoid(z.abs())
    t = (n / 64 + 32) * U
    e1 = gmean((dz * g).abs()) * t + gmean(edz * g.abs())
    e2 = gmean((dz * g * xh).abs()) * (t + 4 * U) + gmean(edz * (g * xh).abs())
    edx = rs * (edz * g.abs() + e1 + xh.abs() * e2 + 8 * U * ((dz * g).abs() + m1.abs() + (xh * m2).abs()))
    tp = (B * S / 64 + 64) * U

    def csum(t):
        return sums(t.reshape(B * S, C))

    dg, db = csum(dz * xh), csum(dz)
    edg = csum((dz * xh).abs()) * (tp + 4 * U) + csum(edz * xh.abs())
    edb = csum(dz.abs()) * tp + csum(edz)
    return (dx, dg, db), (edx + half(dt) * dx.abs() + tiny(dt), edg, edb)


def most(v):
    """The largest of a vector, 256 values at a time (as sums)."""
    while v.numel() > 256:
        n = -(-v.numel() // 256)
        w = v[:1].expand(n * 256).clone()
        w[:v.numel()] = v
        v = w.view(n, 256).amax(1)
    return v.max().item()


def within(got, want, bound):
    """got is within bound of want; a half-precision result of 65520 and more (65504 and half a step)
    rounds to infinity, as the type has it."""
    far = (want.abs() - bound >= 65520) & (got.dtype == torch.float16)
    got = got.double().reshape(want.shape)
    assert torch.equal(got[far], torch.sign(want[far]) * float("inf"))
    got, want, bound = got[~far], want[~far], bound[~far]
    if got.numel():
        assert most((~torch.isfinite(got)).double()) == 0
        off = (got - want).abs().flatten()
        over = most(off - bound.flatten())
        assert over <= 0, f"off by {most(off):.3g}, {over:.3g} more than the bound"
