"""Autograd forms of ops.class_logprobs and ops.distill_loss: what a loss on class scores is built from (the cross entropies of
lib/nets/network.py:319-501 are `-logp` averaged over the rows that carry a label)."""
import torch
from torch.autograd.function import once_differentiable

from .. import ops


class ClassLogProbs(torch.autograd.Function):
    """`ClassLogProbs.apply(score, labels, top, num)` -> (logp, entropy, top_logp, top_class); gradients reach score through logp and
    entropy, the alternatives are reported and carry none.  A training step may be captured into a graph as any of torch's: no eager
    backward graph of the same parameters may be alive then."""

    @staticmethod
    def forward(ctx, score, labels, top=0, num=None):
        logp, entropy, norm, top_logp, top_class = ops.class_logprobs(score, labels, top, num)
        ctx.save_for_backward(score, labels, norm, entropy, num)
        ctx.mark_non_differentiable(top_logp, top_class)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_class

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logp, grad_entropy, *_):
        score, labels, norm, entropy, num = ctx.saved_tensors
        if grad_logp is None and grad_entropy is None:
            return None, None, None, None
        if grad_logp is None:
            grad_logp = torch.zeros_like(grad_entropy)
        return ops.class_logprobs_backward(score, labels, norm, entropy, grad_logp, grad_entropy, num), None, None, None


class DistillLoss(torch.autograd.Function):
    """`DistillLoss.apply(score, kept, classes, temperature, num)` -> loss per row; the teacher's logits get no gradient."""

    @staticmethod
    def forward(ctx, score, kept, classes, temperature=1.0, num=None):
        loss, norm = ops.distill_loss(score, kept, classes, temperature, num)
        ctx.save_for_backward(score, kept, classes, norm, num)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        score, kept, classes, norm, num = ctx.saved_tensors
        return ops.distill_loss_backward(score, kept, classes, norm, grad_loss, ctx.temperature, num), None, None, None, None
