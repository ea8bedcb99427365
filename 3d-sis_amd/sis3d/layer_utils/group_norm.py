"""Autograd form of ops.group_norm."""
import torch
from torch.autograd.function import once_differentiable

from .. import ops


class GroupNormAct(torch.autograd.Function):
    """`GroupNormAct.apply(x, weight, bias, groups, eps, act, offsets)` -> y: ops.group_norm with gradients for x, weight and bias.

    A training step may be captured into a graph as any of torch's: no eager backward graph of the same parameters may be alive then."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps=1e-5, act=None, offsets=None):
        y, mean, rstd = ops.group_norm(x, groups, weight, bias, eps, act=act, offsets=offsets, want_stats=True)
        ctx.save_for_backward(x, weight, bias, mean, rstd, offsets)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd, offsets = ctx.saved_tensors
        try:
            ops._channel_rows(dy.shape, dy.stride(), None if offsets is None else offsets.numel() - 1, "dy")
        except ops._lib.Sis3dError:                 # autograd may hand in any layout (an expanded sum's gradient, a planar one)
            dy = torch.empty_strided(x.shape, ops._last_second(x.shape), dtype=x.dtype, device=x.device).copy_(dy)
        dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, ctx.groups, weight, bias, act=ctx.act, offsets=offsets)
        return dx, dw, db, None, None, None, None
