"""Distillation from a teacher's top logits on the GPU (stes_distill / stes_distill_bwd in include/stes.h): the KL divergence of a
student's class distribution from the teacher's distribution over its k best classes, and its gradient.

    loss = topk_distill_loss(student_logits, idx, val, temperature=2.0)             # for loss.backward()
    loss, dlogits = topk_distill_grad(student_logits, idx, val, temperature=2.0)    # both in one pass over the logits

`idx` and `val` are what `teacher_logits.topk(k)` gives; an index below zero marks an unused place of a frame's list.
"""
from __future__ import annotations

import functools
import math

import torch

from . import lib

_ELEMENT = {torch.bfloat16: 0, torch.float32: 1}


def _refuse(text):
    raise lib.StesError("topk_distill: " + text)


def _flat(t, n):
    """[..., n] -> [M, n] without a copy where the strides allow one row stride, else a contiguous copy."""
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if not t.is_contiguous() and ((n > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < n)):
        t = t.contiguous()
    return t


def _at(t):
    return 0 if t is None else t.data_ptr()


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


@functools.lru_cache(maxsize=256)
def _ws_floats(M, V, k):
    return lib.lib().stes_distill_ws_floats(M, V, k)


def _call(entry, logits, idx, val, weight, temperature, denom, grad_scale=1.0, upstream=None, loss=None, stats=None, d=None, accumulate=False):
    """One call of the library; every tensor [M, ...] with contiguous rows."""
    M, V = logits.shape
    n = 0 if loss is None else _ws_floats(M, V, idx.shape[1])
    ws = torch.empty(n, dtype=torch.float32, device=logits.device) if n else None          # (of this call's own)
    lib.call(entry, lib.pack_distill(
        logits.data_ptr(), _ld(logits), _ELEMENT[logits.dtype], idx.data_ptr(), _ld(idx), idx.dtype == torch.int64,
        val.data_ptr(), _ld(val), _ELEMENT[val.dtype], _at(weight), M, V, idx.shape[1], temperature, denom, grad_scale, _at(upstream),
        _at(loss), _at(stats), _at(d), 0 if d is None else _ld(d), 0 if d is None else _ELEMENT[d.dtype], accumulate, _at(ws), n))


class _Distill(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, idx, val, weight, temperature, denom):
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        stats = torch.empty(logits.shape[0], 2, dtype=torch.float32, device=logits.device)
        _call("stes_distill", logits, idx, val, weight, temperature, denom, loss=loss, stats=stats)
        ctx.save_for_backward(logits, idx, val, weight, stats)
        ctx.scale = (temperature, denom)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        logits, idx, val, weight, stats = ctx.saved_tensors
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if logits.shape[0]:
            with lib.on_device(logits.device):
                _call("stes_distill_bwd", logits, idx, val, weight, *ctx.scale, upstream=up, stats=stats, d=d)
        return d, None, None, None, None, None


def _check(logits, idx, val, weight, temperature, denom):
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in _ELEMENT or logits.dim() < 1:
        _refuse("logits must be a bfloat16 or float32 tensor [..., classes] on the GPU")
    dev, V, lead = logits.device, logits.shape[-1], logits.shape[:-1]
    if V < 1:
        _refuse("no classes")
    if idx.device != dev or idx.dtype not in (torch.int64, torch.int32) or idx.dim() != logits.dim() or idx.shape[:-1] != lead:
        _refuse(f"idx must be int64 or int32 {list(lead)} + [k] on {dev}, got {idx.dtype} {list(idx.shape)} on {idx.device}")
    k = idx.shape[-1]
    if not 1 <= k <= lib.DISTILL_MAX_K:
        _refuse(f"1 to {lib.DISTILL_MAX_K} teacher classes a row, got {k}")
    if val.device != dev or val.dtype not in _ELEMENT or val.shape != idx.shape:
        _refuse(f"val must be float32 or bfloat16 {list(idx.shape)} on {dev}")
    if weight is not None and (weight.device != dev or weight.dtype != torch.float32 or weight.shape != lead):
        _refuse(f"weight must be float32 {list(lead)} on {dev}")
    if torch.is_grad_enabled() and (val.requires_grad or (weight is not None and weight.requires_grad)):
        _refuse("the teacher's logits and the weights are constants: detach them")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        _refuse(f"the temperature lies between 1e-6 and 1e6, got {temperature}")
    s = _flat(logits, V)
    denom = float(max(1, s.shape[0]) if denom is None else denom)
    if not 0.0 < denom < math.inf:
        _refuse(f"the denominator is positive, got {denom}")
    if weight is not None:
        weight = weight.reshape(-1).contiguous()
    return s, _flat(idx, k), _flat(val, k), weight, temperature, denom


def topk_distill_loss(logits, idx, val, temperature=1.0, weight=None, denom=None):
    """tau^2 / denom * sum over rows of weight * KL(P || q): q = softmax(logits / tau) over all classes, P = softmax(val / tau) over
    the listed ones.

    logits  [..., V] bfloat16 or float32, the student's; differentiable (once)
    idx     [..., k] int64 or int32, k <= 64: the classes the teacher rates highest; below zero: an unused place
    val     [..., k] float32 or bfloat16: the teacher's logits of these classes
    weight  [...] float32 or None (ones); rows of weight 0 and rows without a class add nothing, whatever their logits hold
    denom   a number; None: the number of rows
    -> a float32 scalar.  A class listed twice has the sum of its probabilities; an index beyond V makes the result NaN."""
    s, idx, val, weight, temperature, denom = _check(logits, idx, val, weight, temperature, denom)
    with lib.on_device(s.device):
        if s.requires_grad and torch.is_grad_enabled():
            loss = _Distill.apply(s, idx, val, weight, temperature, denom)
            lib.guard_leaves(loss.grad_fn)
            return loss
        loss = torch.empty((), dtype=torch.float32, device=s.device)
        _call("stes_distill", s, idx, val, weight, temperature, denom, loss=loss)
    return loss


def topk_distill_grad(logits, idx, val, temperature=1.0, weight=None, denom=None, grad_scale=1.0, out=None, accumulate=False):
    """The loss of topk_distill_loss and grad_scale times its gradient in ONE pass over the logits, for training steps without autograd.

    out         where the gradient goes: bfloat16 or float32 [..., V] (any row stride), None: a new tensor of the logits' type; it shares
                no memory with what the call reads
    accumulate  add to `out` instead of writing it
    -> (loss, gradient)"""
    s, idx, val, weight, temperature, denom = _check(logits, idx, val, weight, temperature, denom)
    if out is None:
        if accumulate:
            _refuse("accumulate adds to out")
        out = torch.empty(logits.shape, dtype=logits.dtype, device=s.device)
    elif out.device != s.device or out.dtype not in _ELEMENT or out.shape != logits.shape or (out.requires_grad and torch.is_grad_enabled()):
        _refuse(f"out must be float32 or bfloat16 {list(logits.shape)} on {s.device}, without gradients")
    try:
        d = out if out.dim() == 2 else out.view(-1, out.shape[-1])
    except RuntimeError:
        _refuse("rows of out must be one stride apart")
    if not d.is_contiguous() and ((d.shape[1] > 1 and d.stride(1) != 1) or (d.shape[0] > 1 and d.stride(0) < d.shape[1])):
        _refuse("rows of out must be contiguous and not overlap")
    with lib.on_device(s.device):
        loss = torch.empty((), dtype=torch.float32, device=s.device)
        _call("stes_distill", s, idx, val, weight, temperature, denom, float(grad_scale), loss=loss, d=d, accumulate=bool(accumulate))
        lib.written(out)
    return loss, out
