"""Autograd entry points of the group-norm and 8-bit checkpoint kernels (ops/kernels.py).

``group_norm_act`` and ``conv1x1`` take tensors as a module has them (any strides, any device, channels
first in shape) and hand channels-last operands to the kernels; a ``channels_last`` tensor is not
copied.  Outputs are channels last, and code may write into them.  On a CPU tensor they are the plain torch operations, with exact gradients.
"""
import contextlib
from typing import Tuple, Union

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import kernels as K

ACTS = {"none": K.GN_NONE, "relu": K.GN_RELU, "relu6": K.GN_RELU6, "silu": K.GN_SILU}
_PLAIN = {"none": lambda y: y, "relu": F.relu, "relu6": F.relu6, "silu": F.silu}


def _rows(x):
    """[B, C, ...] -> [B, ..., C], contiguous and 16-byte aligned (no copy of a channels-last tensor)."""
    x = x.movedim(1, -1).contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _like_rows(rows, C):
    """An output of C channels for channels-last rows [B, ..., n]: ([B, C, ...], its [B, ..., C] alias). The first is
    the tensor itself and the alias a view of it: autograd refuses in-place code behind an operator that returns a
    view of its own making."""
    shape, stride, n = (*rows.shape[:-1], C), [], 1
    for d in reversed(shape):
        stride.insert(0, n)
        n *= max(d, 1)
    y = torch.empty_strided((shape[0], C, *shape[1:-1]), (stride[0], 1, *stride[1:-1]), dtype=rows.dtype, device=rows.device)
    return y, y.movedim(1, -1)


def _vec(t):
    """A per-channel parameter as the kernels take it: fp32, contiguous, aligned."""
    if t is None:
        return None
    t = t.detach().to(torch.float32).contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _on(t):
    """The tensor's device as the current one (the launch goes to its current stream)."""
    return torch.cuda.device(t.device) if t.is_cuda else contextlib.nullcontext()


def _codes(M, C, device):
    return (torch.empty(M, C, dtype=torch.uint8, device=device),
            torch.empty(M, K.mx8_blocks(C), dtype=torch.uint8, device=device))


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, ckpt8, grad):
        with _on(x):
            xl = _rows(x)
            B, C = xl.shape[0], xl.shape[-1]
            S = xl.numel() // (B * C) if B else 0
            w, b = _vec(weight), _vec(bias)
            y, yl = _like_rows(xl, C)
            mean = torch.empty(B, groups, dtype=torch.float32, device=x.device)
            rstd = torch.empty_like(mean)
            keep = ckpt8 and grad and any(ctx.needs_input_grad[:3])
            q, qs = _codes(B * S, C, x.device) if keep else (None, None)
            K.gn_fwd(xl, w, b, yl, mean, rstd, B, S, C, groups, eps=eps, act=act, q=q, qs=qs, as_ckpt8=ckpt8)
        ctx.save_for_backward(None if keep else xl, q, qs, w, b, mean, rstd)
        ctx.sizes = (B, S, C, groups, act)
        ctx.dtypes = (None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xl, q, qs, w, b, mean, rstd = ctx.saved_tensors
        B, S, C, groups, act = ctx.sizes
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        with _on(dy):
            dyl = _rows(dy)
            dx = torch.empty_like(dyl)
            dgb = torch.empty(2, C, dtype=torch.float32, device=dy.device) if params else None
            K.gn_bwd(dyl, xl, w, b, mean, rstd, dx, dgb, B, S, C, groups, act=act, q=q, qs=qs)
        dw = dgb[0].to(ctx.dtypes[0]) if ctx.needs_input_grad[1] else None
        db = dgb[1].to(ctx.dtypes[1]) if ctx.needs_input_grad[2] else None
        return dx.movedim(-1, 1) if ctx.needs_input_grad[0] else None, dw, db, None, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none", ckpt8=False):
    """act(group_norm(x)) of [B, C, ...] with its gradients.  act: none, relu, relu6 or silu.  On the
    GPU x is bf16, fp16 or fp32; weight and bias are [C] of any floating type.
    ``ckpt8``: the backward pass keeps x as its 8-bit checkpoint (kernels.mx8_pack) instead of as it
    is, and its gradients are those of the values that stands for.  Without gradients none is made, and
    the result has the same bits."""
    if act not in ACTS:
        raise ValueError(f"group_norm_act: unknown activation {act!r}; available: {sorted(ACTS)}")
    if x.dim() < 2:
        raise ValueError("group_norm_act: x must be [B, C, ...]")
    C = x.shape[1]
    if C < 1 or groups < 1 or C % groups:
        raise ValueError(f"group_norm_act: {groups} groups do not divide {C} channels")
    for t, nm in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != (C,) or t.device != x.device):
            raise ValueError(f"group_norm_act: {nm} must be [{C}] on {x.device}, got {list(t.shape)} on {t.device}")
    if not x.is_cuda:
        return _PLAIN[act](F.group_norm(x, groups, weight, bias, eps))
    # needs_input_grad does not know of no_grad, and gradients are off within forward
    return _GroupNormAct.apply(x, weight, bias, groups, eps, ACTS[act], ckpt8, torch.is_grad_enabled())


class GroupNormAct(nn.Module):
    """Group norm and an activation in one pass; parameters ``weight`` and ``bias`` as nn.GroupNorm's."""

    def __init__(self, num_groups: int, num_channels: int, act: str = "none", eps: float = 1e-5, ckpt8: bool = False):
        super().__init__()
        if num_channels < 1 or num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"GroupNormAct: {num_groups} groups do not divide {num_channels} channels")
        if act not in ACTS:
            raise ValueError(f"GroupNormAct: unknown activation {act!r}; available: {sorted(ACTS)}")
        self.num_groups, self.num_channels, self.act, self.eps, self.ckpt8 = num_groups, num_channels, act, eps, ckpt8
        self.weight = nn.Parameter(torch.ones(num_channels))
        self.bias = nn.Parameter(torch.zeros(num_channels))

    def forward(self, x):
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, self.ckpt8)

    def extra_repr(self):
        return f"{self.num_groups}, {self.num_channels}, act={self.act}, eps={self.eps}, ckpt8={self.ckpt8}"


class _Conv1x1(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, dtype, grad):
        with _on(x):
            xl = _rows(x.to(dtype))
            N, C = weight.shape[:2]
            M = xl.numel() // C
            w = weight.detach().reshape(N, C).to(dtype)
            y, yl = _like_rows(xl, N)
            if bias is None:
                torch.mm(xl.view(M, C), w.t(), out=yl.view(M, N))
            else:   # the bias joins the product's fp32 sums: one rounding
                torch.addmm(bias.detach().to(dtype), xl.view(M, C), w.t(), out=yl.view(M, N))
            q = qs = None
            if grad and ctx.needs_input_grad[1]:
                q, qs = _codes(M, C, x.device)
                K.mx8_pack(xl, q, qs, M, C)
        ctx.save_for_backward(w if ctx.needs_input_grad[0] else None, q, qs)
        ctx.sizes = (M, N, C, x.dtype, weight.shape, weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, q, qs = ctx.saved_tensors
        M, N, C, xdt, wshape, wdt, bdt = ctx.sizes
        dx = dw = db = None
        with _on(dy):
            dyl = _rows(dy)
            if ctx.needs_input_grad[0]:
                dx = (dyl.view(M, N) @ w).view(*dyl.shape[:-1], C).movedim(-1, 1).to(xdt)
            if ctx.needs_input_grad[1]:
                dw = torch.empty(N, C, dtype=torch.float32, device=dy.device)
                db = torch.empty(N, dtype=torch.float32, device=dy.device) if ctx.needs_input_grad[2] else None
                K.mx8_wgrad(dyl, q, qs, dw, M, N, C, db=db)
                dw = dw.view(wshape).to(wdt)
            elif ctx.needs_input_grad[2]:
                db = torch.empty(N, dtype=torch.float32, device=dy.device)
                z = torch.zeros(M, 8, dtype=torch.uint8, device=dy.device)   # no input was kept: beside a product with zeros
                K.mx8_wgrad(dyl, z, z.view(-1)[:M].view(M, 1), torch.empty(N, 8, dtype=torch.float32, device=dy.device),
                            M, N, 8, db=db)
        return dx, dw, None if db is None else db.to(bdt), None, None


def conv1x1(x, weight, bias=None, stride=1):
    """1x1 convolution of [B, C, H, W] (weight [N, C, 1, 1]; stride one number or one a direction) whose
    backward pass keeps its input as the 8-bit checkpoint (kernels.mx8_pack): dW and db come from
    kernels.mx8_wgrad.  On the GPU in bf16 or fp16 (the input's type, or autocast's); any other call,
    in fp32 above all, is the plain convolution, which keeps its input as it is.  Where no gradient is
    wanted no checkpoint is made."""
    stride = tuple(stride) if isinstance(stride, (tuple, list)) else (stride,)
    stride = stride * 2 if len(stride) == 1 else stride
    if len(stride) != 2 or min(stride) < 1:
        raise ValueError(f"conv1x1: stride {stride} must be a positive number or two")
    if x.dim() != 4 or weight.dim() != 4 or tuple(weight.shape[2:]) != (1, 1) or weight.shape[1] != x.shape[1]:
        raise ValueError(f"conv1x1: x [B, C, H, W] and weight [N, C, 1, 1], got {tuple(x.shape)}, {tuple(weight.shape)}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != x.device):
        raise ValueError(f"conv1x1: bias must be [{weight.shape[0]}] on {x.device}, got {list(bias.shape)} on {bias.device}")
    cast = x.is_cuda and x.dtype != torch.float64 and torch.is_autocast_enabled("cuda")   # autocast leaves fp64 alone
    dtype = torch.get_autocast_dtype("cuda") if cast else x.dtype
    if not x.is_cuda or dtype not in (torch.bfloat16, torch.float16) or x.numel() == 0:
        return F.conv2d(x, weight, bias, stride)
    if stride != (1, 1):
        x = x[:, :, ::stride[0], ::stride[1]]
    return _Conv1x1.apply(x, weight, bias, dtype, torch.is_grad_enabled())


class Conv1x1Ckpt8(nn.Conv2d):
    """nn.Conv2d of kernel size 1 (no padding, no groups) through :func:`conv1x1`."""

    def __init__(self, cin: int, cout: int, stride: Union[int, Tuple[int, int]] = 1, bias: bool = False):
        super().__init__(cin, cout, 1, stride, bias=bias)

    def forward(self, x):
        return conv1x1(x, self.weight, self.bias, self.stride)
