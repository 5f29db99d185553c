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
