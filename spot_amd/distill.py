"""Distillation from a teacher's top logits on the GPU (stes_distill / stes_distill_bwd in include/stes.h): the KL divergence of a
student's class distribution from the teacher's distribution over its k best classes, and its gradient.

    loss = topk_distill_loss(student_logits, idx, val, temperature=2.0)             # for loss.backward()
    loss, dlogits = topk_distill_grad(student_logits, idx, val, temperature=2.0)    # both in one pass over the logits

`idx` and `val` are what `teacher_logits.topk(k)` gives; an index below zero marks an unused place of a frame's list.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import lib

_ELEMENT = {torch.bfloat16: 0, torch.float32: 1}


def _need(ok, text):
    if not ok:
        raise lib.StesError("topk_distill: " + text)


def _flat(t, n):
    """[..., n] -> [M, n] without a copy where the strides allow one row stride, else a contiguous copy."""
    t = t.reshape(-1, n) if t.dim() != 2 else t
    if (n > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < n):
        t = t.contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _args(logits, idx, val, weight, temperature, denom):
    """-> (argument block, the tensors it points at); logits is [M, V], rows contiguous."""
    M, V = logits.shape
    a = lib.DistillArgs()
    k = idx.shape[1]
    a.M, a.V, a.k = M, V, k
    a.logits, a.ld, a.f32 = logits.data_ptr(), _ld(logits), _ELEMENT[logits.dtype]
    a.idx, a.ld_idx, a.idx_i64 = idx.data_ptr(), _ld(idx), int(idx.dtype == torch.int64)
    a.val, a.ld_val, a.val_f32 = val.data_ptr(), _ld(val), _ELEMENT[val.dtype]
    if weight is not None:
        a.weight = weight.data_ptr()
    a.temperature, a.denom, a.grad_scale = temperature, denom, 1.0
    return a


def _workspace(a, dev):
    n = lib.lib().stes_distill_ws_floats(a.M, a.V)
    ws = torch.empty(n, dtype=torch.float32, device=dev)
    a.ws, a.ws_floats = ws.data_ptr(), n
    return ws


class _Distill(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, idx, val, weight, temperature, denom):
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        stats = torch.empty(logits.shape[0], 2, dtype=torch.float32, device=logits.device)
        a = _args(logits, idx, val, weight, temperature, denom)
        _ws = _workspace(a, logits.device)
        a.loss, a.stats = loss.data_ptr(), stats.data_ptr()
        lib.call("stes_distill", C.byref(a))
        ctx.save_for_backward(logits, idx, val, weight, stats)
        ctx.scale = (temperature, denom)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        logits, idx, val, weight, stats = ctx.saved_tensors
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if logits.shape[0]:
            with torch.cuda.device(logits.device):
                up = up.to(torch.float32)
                a = _args(logits, idx, val, weight, *ctx.scale)
                a.stats, a.upstream = stats.data_ptr(), up.data_ptr()
                a.dlogits, a.ld_d, a.d_f32 = d.data_ptr(), _ld(d), _ELEMENT[d.dtype]
                lib.call("stes_distill_bwd", C.byref(a))
        return d, None, None, None, None, None


def _check(logits, idx, val, weight, temperature, denom):
    _need(isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _ELEMENT and logits.dim() >= 1,
          "logits must be a bfloat16 or float32 tensor [..., classes] on the GPU")
    dev, V, lead = logits.device, logits.shape[-1], tuple(logits.shape[:-1])
    _need(V >= 1, "no classes")
    _need(idx.device == dev and idx.dtype in (torch.int64, torch.int32) and idx.dim() == logits.dim() and tuple(idx.shape[:-1]) == lead,
          f"idx must be int64 or int32 {list(lead)} + [k] on {dev}, got {idx.dtype} {list(idx.shape)} on {idx.device}")
    k = idx.shape[-1]
    _need(1 <= k <= lib.DISTILL_MAX_K, f"1 to {lib.DISTILL_MAX_K} teacher classes a row, got {k}")
    _need(val.device == dev and val.dtype in _ELEMENT and val.shape == idx.shape, f"val must be float32 or bfloat16 {list(idx.shape)} on {dev}")
    _need(not (torch.is_grad_enabled() and val.requires_grad), "the teacher's logits are constants: detach val")
    if weight is not None:
        _need(weight.device == dev and weight.dtype == torch.float32 and tuple(weight.shape) == lead, f"weight must be float32 {list(lead)} on {dev}")
        _need(not (torch.is_grad_enabled() and weight.requires_grad), "weights are constants: detach weight")
        weight = weight.reshape(-1).contiguous()
    temperature = float(temperature)
    _need(0.0 < temperature < float("inf"), f"the temperature is positive, got {temperature}")
    s = _flat(logits, V)
    denom = float(max(1, s.shape[0]) if denom is None else denom)
    _need(0.0 < denom < float("inf"), f"the denominator is positive, got {denom}")
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
    with torch.cuda.device(s.device):
        if torch.is_grad_enabled() and s.requires_grad:
            loss = _Distill.apply(s, idx, val, weight, temperature, denom)
            lib.guard_leaves(loss.grad_fn)
            return loss
        loss = torch.empty((), dtype=torch.float32, device=s.device)
        a = _args(s, idx, val, weight, temperature, denom)
        _ws = _workspace(a, s.device)
        a.loss = loss.data_ptr()
        lib.call("stes_distill", C.byref(a))
    return loss


def topk_distill_grad(logits, idx, val, temperature=1.0, weight=None, denom=None, grad_scale=1.0, out=None, accumulate=False):
    """The loss of topk_distill_loss and grad_scale times its gradient in ONE pass over the logits, for training steps without autograd.

    out         where the gradient goes: bfloat16 or float32 [..., V] (any row stride), None: a new tensor of the logits' type
    accumulate  add to `out` instead of writing it
    -> (loss, gradient)"""
    s, idx, val, weight, temperature, denom = _check(logits.detach(), idx, val, weight, temperature, denom)
    _need(not accumulate or out is not None, "accumulate adds to out")
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=s.device)
    else:
        _need(out.device == s.device and out.dtype in _ELEMENT and out.shape == logits.shape, f"out must be float32 or bfloat16 {list(logits.shape)} on {s.device}")
    d = out if out.dim() == 2 else out.view(-1, out.shape[-1])
    _need((d.shape[1] <= 1 or d.stride(1) == 1) and (d.shape[0] <= 1 or d.stride(0) >= d.shape[1]), "rows of out must be contiguous and not overlap")
    with torch.cuda.device(s.device):
        loss = torch.empty((), dtype=torch.float32, device=s.device)
        a = _args(s, idx, val, weight, temperature, denom)
        _ws = _workspace(a, s.device)
        a.grad_scale, a.loss = float(grad_scale), loss.data_ptr()
        a.dlogits, a.ld_d, a.d_f32, a.accumulate = d.data_ptr(), _ld(d), _ELEMENT[d.dtype], int(accumulate)
        lib.call("stes_distill", C.byref(a))
    return loss, out
