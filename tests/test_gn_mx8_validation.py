"""Refusals of the group-norm and 8-bit checkpoint wrappers: raised on the host before any launch."""
import pytest
import torch

import pgdist  # noqa: F401
from pgdist.ops import kernels as K

B, S, C, G = 2, 6, 32, 4
BF, U8 = torch.bfloat16, torch.uint8


def fwd_args():
    return dict(x=torch.zeros(B, S, C, dtype=BF), gamma=torch.ones(C), beta=torch.zeros(C), y=torch.zeros(B, S, C, dtype=BF),
                mean=torch.zeros(B, G), rstd=torch.zeros(B, G), B=B, S=S, C=C, G=G, act=K.GN_RELU,
                q=torch.zeros(B * S, C, dtype=U8), qs=torch.zeros(B * S, 1, dtype=U8))


def bwd_args():
    a = fwd_args()
    return dict(dy=a["x"], x=a["x"].clone(), gamma=a["gamma"], beta=a["beta"], mean=a["mean"], rstd=a["rstd"],
                dx=a["y"], dgb=torch.zeros(2, C), B=B, S=S, C=C, G=G, act=K.GN_RELU)


FWD = [(dict(G=5), ValueError, "divide"), (dict(G=0), ValueError, "divide"), (dict(S=-1), ValueError, "divide"),
       (dict(act=7), ValueError, "activation"), (dict(eps=0.0), ValueError, "eps"), (dict(eps=float("nan")), ValueError, "eps"),
       (dict(q=None), ValueError, "both"), (dict(qs=None), ValueError, "both"),
       (dict(x=torch.zeros(B, S, C, dtype=torch.int32)), TypeError, "bf16"),
       (dict(y=torch.zeros(B, S, C)), TypeError, "y"), (dict(y=torch.zeros(B, S, C - 1, dtype=BF)), ValueError, "y"),
       (dict(x=torch.zeros(B, C, S, dtype=BF).transpose(1, 2)), ValueError, "contiguous"),
       (dict(x=torch.zeros(B * S * C + 1, dtype=BF)[1:]), ValueError, "aligned"),
       (dict(gamma=torch.ones(C, dtype=BF)), TypeError, "gamma"), (dict(beta=torch.ones(C + 1)), ValueError, "beta"),
       (dict(mean=torch.zeros(B, C)), ValueError, "mean"), (dict(rstd=torch.zeros(B, G, dtype=torch.float64)), TypeError, "rstd"),
       (dict(q=torch.zeros(B * S, C)), TypeError, "q"), (dict(qs=torch.zeros(B * S, 2, dtype=U8)), ValueError, "qs"),
       (dict(), ValueError, "device tensor")]


@pytest.mark.parametrize("change,error,word", FWD)
def test_gn_fwd_refuses(change, error, word):
    with pytest.raises(error, match=word):
        K.gn_fwd(**{**fwd_args(), **change})


def test_gn_fwd_refuses_shared_memory():
    a = fwd_args()
    with pytest.raises(ValueError, match="overlaps"):
        K.gn_fwd(**{**a, "y": a["x"]})
    with pytest.raises(ValueError, match="overlaps"):
        K.gn_fwd(**{**a, "rstd": a["mean"]})
    big = torch.zeros(B * S * C + 64, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        K.gn_fwd(**{**a, "x": big[:B * S * C], "y": big[64:]})


BWD = [(dict(x=None), ValueError, "either"), (dict(q=torch.zeros(B * S, C, dtype=U8)), ValueError, "either"),
       (dict(q=torch.zeros(B * S, C, dtype=U8), qs=torch.zeros(B * S, 1, dtype=U8)), ValueError, "either"),
       (dict(x=None, q=torch.zeros(B * S, C - 1, dtype=U8), qs=torch.zeros(B * S, 1, dtype=U8)), ValueError, "q"),
       (dict(dx=torch.zeros(B, S, C)), TypeError, "dx"), (dict(dgb=torch.zeros(C)), ValueError, "dgb"),
       (dict(x=torch.zeros(B, S, C)), TypeError, "x"), (dict(act=-1), ValueError, "activation"),
       (dict(G=3), ValueError, "divide"), (dict(), ValueError, "device tensor")]


@pytest.mark.parametrize("change,error,word", BWD)
def test_gn_bwd_refuses(change, error, word):
    with pytest.raises(error, match=word):
        K.gn_bwd(**{**bwd_args(), **change})


def test_gn_bwd_refuses_in_place():
    a = bwd_args()
    for name in ("dy", "x"):
        with pytest.raises(ValueError, match="overlaps"):
            K.gn_bwd(**{**a, "dx": a[name]})


def test_mx8_refuses():
    x, q, qs = torch.zeros(4, 40, dtype=BF), torch.zeros(4, 40, dtype=U8), torch.zeros(4, 2, dtype=U8)
    for f, args in ((K.mx8_pack, lambda x=x, q=q, qs=qs, M=4, C=40: (x, q, qs, M, C)),
                    (K.mx8_unpack, lambda x=x, q=q, qs=qs, M=4, C=40: (q, qs, x, M, C))):
        for kw, error in ((dict(x=x.double()), TypeError), (dict(q=q.float()), TypeError), (dict(M=5), ValueError),
                          (dict(C=0), ValueError), (dict(M=-1), ValueError), (dict(qs=qs[:, :1].contiguous()), ValueError),
                          (dict(x=x[:, ::2]), ValueError), (dict(), ValueError)):
            with pytest.raises(error):
                f(*args(**kw))
    raw = torch.zeros(1024, dtype=U8)
    with pytest.raises(ValueError, match="overlaps"):
        K.mx8_pack(raw[:320].view(BF).view(4, 40), raw[160:320].view(4, 40), qs, 4, 40)


def test_mx8_wgrad_refuses():
    a = dict(dy=torch.zeros(4, 8, dtype=BF), q=torch.zeros(4, 40, dtype=U8), qs=torch.zeros(4, 2, dtype=U8),
             grad=torch.zeros(8, 40), M=4, N=8, K=40, db=torch.zeros(8))
    for kw, error, word in ((dict(dy=torch.zeros(4, 8)), TypeError, "bf16 or fp16"), (dict(N=7), ValueError, "dy"),
                            (dict(K=0), ValueError, "positive"), (dict(M=-1), ValueError, "M="),
                            (dict(grad=torch.zeros(8, 40, dtype=BF)), TypeError, "grad"),
                            (dict(db=torch.zeros(9)), ValueError, "db"), (dict(qs=torch.zeros(4, 1, dtype=U8)), ValueError, "qs"),
                            (dict(M=1 << 31), ValueError, "below"), (dict(), ValueError, "device tensor")):
        with pytest.raises(error, match=word):
            K.mx8_wgrad(**{**a, **kw})
    with pytest.raises(ValueError, match="overlaps"):
        K.mx8_wgrad(**{**a, "db": a["grad"].view(-1)[:8]})


def test_sizes_of_workspaces_are_checked():
    for args, error in (((-1, 4, 32, 4, BF), ValueError), ((1, 4, 0, 1, BF), ValueError), ((1, 4, 32, 0, BF), ValueError),
                        ((1, 4, 32, 5, BF), ValueError), ((1, 4, 1 << 30, 4, BF), ValueError),
                        ((1, 4, 32, 4, torch.float64), TypeError)):
        with pytest.raises(error):
            K.gn_workspace(*args)
    for args in ((4, 0, 40), (4, 8, 0), (-1, 8, 40), (4, 1 << 31, 40)):
        with pytest.raises(ValueError):
            K.mx8_wgrad_workspace(*args)
    assert K.gn_workspace(0, 4, 32, 4, BF) == 0 and K.mx8_wgrad_workspace(0, 8, 40) == 0


@pytest.mark.parametrize("eps", [1e-45, float("inf")])
def test_gn_fwd_refuses_an_eps_that_fp32_does_not_hold(eps):
    with pytest.raises(ValueError, match="eps"):
        K.gn_fwd(**{**fwd_args(), "eps": eps})


def test_modules_refuse_no_channels():
    from pgdist.ops import nn as N
    with pytest.raises(ValueError):
        N.GroupNormAct(1, 0)
    with pytest.raises(ValueError):
        N.group_norm_act(torch.zeros(2, 0, 3, 3), 1)


def test_blocks():
    assert [K.mx8_blocks(c) for c in (1, 32, 33, 144)] == [1, 1, 2, 5]
