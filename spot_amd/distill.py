"""Distillation from a teacher's top logits on the GPU (stes_distill / stes_distill_bwd in include/stes.h): the KL divergence of a
student's class distribution from the teacher's distribution over its k best classes, and its gradient.

    loss = topk_distill_loss(student_logits, idx, val, temperature=2.0)             # for loss.backward()
    loss, dlogits = topk_distill_grad(student_logits, idx, val, temperature=2.0)    # both in one pass over the logits

`idx` and `val` are what `teacher_logits.topk(k)` gives; an index below zero marks an unused place of a frame's list.  Neither call can be
traced (torch.jit.trace, make_fx).
"""
from __future__ import annotations

from . import lib


def topk_distill_loss(logits, idx, val, temperature=1.0, weight=None, denom=None):
    """tau^2 / denom * sum over rows of weight * KL(P || q): q = softmax(logits / tau) over all classes, P = softmax(val / tau) over
    the listed ones.

    logits  [..., V] bfloat16 or float32, the student's; differentiable (once)
    idx     [..., k] int64 or int32, k <= 64: the classes the teacher rates highest; below zero: an unused place
    val     [..., k] float32 or bfloat16: the teacher's logits of these classes
    weight  [...] float32 or None (ones); rows of weight 0 and rows without a class add nothing, whatever their logits hold
    denom   a number; None: the number of rows
    -> a float32 scalar.  A class listed twice has the sum of its probabilities; an index beyond V makes the result NaN."""
    return lib.native_call("distill_kernel", lib.native().topk_distill_loss, logits, idx, val, temperature, weight, denom)


def topk_distill_grad(logits, idx, val, temperature=1.0, weight=None, denom=None, grad_scale=1.0, out=None, accumulate=False):
    """The loss of topk_distill_loss and grad_scale times its gradient in ONE pass over the logits, for training steps without autograd.

    out         where the gradient goes: bfloat16 or float32 [..., V] (any row stride), None: a new tensor of the logits' type; it shares
                no memory with what the call reads
    accumulate  add to `out` instead of writing it
    -> (loss, gradient)"""
    return lib.native_call("distill_kernel", lib.native().topk_distill_grad, logits, idx, val, temperature, weight, denom, grad_scale, out, accumulate)
