"""Group norm and 8-bit checkpoints as programs call them: in-place code behind them, evaluation, odd arguments,
the ends of their ranges."""
import pytest
import torch

import gn_oracle as O
from pgdist.ops import kernels as K
from pgdist.ops import nn as N

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("layout", ["channels_last", "contiguous", "rows"])
@pytest.mark.parametrize("op", ["norm", "norm_ckpt8", "conv"])
def test_in_place_code_behind_an_output(op, layout):
    """relu_ and += on an output give the bits and gradients that the same code gives out of place."""
    if op == "conv" and layout == "rows":
        pytest.skip("a 1x1 convolution takes images")
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
