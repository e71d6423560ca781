"""Gated linear recurrence over sequences of any length on the GPU: the minGRU cell (reference model/min_gru.py:76-92) for whole
videos, frame streams and ragged batches, differentiable (stes_gated_scan_fwd / _bwd in include/stes.h).

    h, last = gated_scan(pre)                                    # [B, T, 2H] -> [B, T, H], fp32 [B, H]
    h, last = gated_scan(pre, h0=last)                           # the next frames of the same sequences
    gated_scan(pre, h0=state, state_out=state)                   # the same, the state updated in place
"""
from __future__ import annotations

import ctypes as C

import torch

from . import lib

_ELEMENT = {torch.bfloat16: 0, torch.float32: 1}


def _need(ok, text):
    if not ok:
        raise lib.StesError("gated_scan: " + text)


def _rows(t, B, H, name):
    """Stride between the rows of a [B, H] fp32 tensor whose rows are contiguous."""
    _need(t.dtype == torch.float32 and tuple(t.shape) == (B, H), f"{name} must be float32 [{B}, {H}], got {t.dtype} {list(t.shape)}")
    _need(H <= 1 or t.stride(1) == 1, f"rows of {name} must be contiguous")
    _need(B <= 1 or t.stride(0) >= H, f"rows of {name} must not overlap")
    return t.stride(0) if B > 1 else max(H, 1)


def _frames(t, width, name):
    """(frame stride, sequence stride) of a [B, T, width] tensor whose last dimension is contiguous."""
    B, T = t.shape[0], t.shape[1]
    _need(width <= 1 or t.stride(2) == 1, f"the last dimension of {name} must be contiguous")
    ld = t.stride(1) if T > 1 else width
    return ld, t.stride(0) if B > 1 else 0


def _apart(t, width):
    """Whether the rows of a [B, T, width] tensor with a contiguous last dimension are apart: frames within sequences or the reverse."""
    inner, outer = sorted((t.stride(i), t.shape[i]) if t.shape[i] > 1 else (0, 1) for i in (0, 1))
    if inner[1] > 1 and inner[0] < width:
        return False
    return outer[1] == 1 or outer[0] >= inner[0] * (inner[1] - 1) + width


def _tidy(t, width):
    """`t` itself where the kernels take its strides, else a contiguous copy (an expanded or transposed gradient)."""
    if (width <= 1 or t.stride(2) == 1) and (t.shape[1] <= 1 or t.stride(1) >= width) and (t.shape[0] <= 1 or t.stride(0) >= 0):
        return t
    return t.contiguous()


def _args(pre, h0, lengths, reverse):
    B, T, W = pre.shape
    H = W // 2
    a = lib.GatedScanArgs()
    a.B, a.T, a.H, a.f32, a.reverse = B, T, H, _ELEMENT[pre.dtype], int(reverse)
    a.pre = pre.data_ptr()
    a.ld_pre, a.bs_pre = _frames(pre, W, "pre")
    if h0 is not None:
        a.h0 = h0.data_ptr()
        a.bs_h0 = 0 if h0.dim() == 1 else _rows(h0, B, H, "h0")
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    need = lib.lib().stes_gated_scan_ws_bytes(B, T, H)
    ws = None
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=pre.device)
        a.ws, a.ws_bytes = ws.data_ptr(), need
    return a, ws


def _forward(pre, h0, lengths, reverse, out, state_out, keep_states):
    B, T, W = pre.shape
    H = W // 2
    h = torch.empty(B, T, H, dtype=pre.dtype, device=pre.device) if out is None else out
    last = torch.empty(B, H, dtype=torch.float32, device=pre.device) if state_out is None else state_out
    states = None
    if keep_states:
        states = torch.empty(B, -(-T // lib.SCAN_BLOCK), H, dtype=torch.float32, device=pre.device)
    if B and H:
        a, _ws = _args(pre, h0, lengths, reverse)
        a.h = h.data_ptr()
        a.ld_h, a.bs_h = _frames(h, H, "out")
        a.h_last, a.bs_hl = last.data_ptr(), _rows(last, B, H, "state_out")
        a.states = lib.ptr(states)
        lib.call("stes_gated_scan_fwd", C.byref(a))
    return h, last, states


class _GatedScan(torch.autograd.Function):

    @staticmethod
    def forward(ctx, pre, h0, lengths, reverse):
        ctx.set_materialize_grads(False)
        h, last, states = _forward(pre, h0, lengths, reverse, None, None, True)
        ctx.save_for_backward(pre, lengths, states)
        ctx.reverse = reverse
        ctx.h0_dim = 0 if h0 is None or not ctx.needs_input_grad[1] else h0.dim()
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        pre, lengths, states = ctx.saved_tensors
        B, T, W = pre.shape
        H = W // 2
        dev = pre.device
        dpre = torch.empty(B, T, W, dtype=pre.dtype, device=dev)
        dh0 = torch.empty(B, H, dtype=torch.float32, device=dev) if ctx.h0_dim else None
        total = torch.empty(H, dtype=torch.float32, device=dev) if ctx.h0_dim == 1 else None
        if H and (B or total is not None):
            with torch.cuda.device(dev):
                a, _ws = _args(pre, None, lengths, ctx.reverse)
                a.states = states.data_ptr()
                if dh is not None:
                    dh = _tidy(dh, H)
                    a.dh = dh.data_ptr()
                    a.ld_dh, a.bs_dh = _frames(dh, H, "dh")
                if dlast is not None:
                    dlast = dlast.contiguous()
                    a.dh_last, a.bs_dhl = dlast.data_ptr(), H
                a.dpre, a.ld_dpre, a.bs_dpre = dpre.data_ptr(), W, T * W
                a.dh0, a.dh0_sum = lib.ptr(dh0), lib.ptr(total)
                lib.call("stes_gated_scan_bwd", C.byref(a))
        return dpre, (total if ctx.h0_dim == 1 else dh0), None, None


def gated_scan(pre, h0=None, lengths=None, reverse=False, out=None, state_out=None):
    """h_t = (1 - z_t) h_{t-1} + z_t c_t with z = sigmoid(pre[..., :H]) and c = pre[..., H:], along the frames of every sequence.

    pre      [B, T, 2H] bfloat16 or float32 on the GPU; the last dimension contiguous, any strides between frames and sequences
    h0       initial states: float32 [B, H], float32 [H] (one for the whole batch) or None (zeros)
    lengths  int32 [B] on the same device (values are clamped to [0, T]) or None: frames from a sequence's length on are not looked at,
             their h (and their gradients) are zero
    reverse  from a sequence's last frame to its first
    out, state_out (without gradients only): where h [B, T, H] and the final states float32 [B, H] go; state_out may be h0
    -> h [B, T, H] in pre's type and the states after the last step, float32 [B, H] (h0 where a sequence is empty)

    Differentiable (once) in pre and h0, from h and from the final states.  T = 0 and T = 1 are calls like any other."""
    _need(isinstance(pre, torch.Tensor) and pre.is_cuda and pre.dim() == 3 and pre.dtype in _ELEMENT,
          "pre must be a bfloat16 or float32 tensor [B, T, 2H] on the GPU")
    B, T, W = pre.shape
    _need(W % 2 == 0, f"the last dimension of pre holds gates and candidates and is even, got {W}")
    H, dev = W // 2, pre.device
    _need(W <= 1 or pre.stride(2) == 1, "the last dimension of pre must be contiguous")
    _need(T <= 1 or pre.stride(1) >= W, "frames of pre must not overlap")
    if h0 is not None:
        _need(h0.device == dev and h0.dtype == torch.float32 and tuple(h0.shape) in ((B, H), (H,)),
              f"h0 must be float32 [{B}, {H}] or [{H}] on {dev}, got {h0.dtype} {list(h0.shape)} on {h0.device}")
        if h0.dim() == 1:
            _need(H <= 1 or h0.stride(0) == 1, "h0 must be contiguous")
        elif (H > 1 and h0.stride(1) != 1) or (B > 1 and h0.stride(0) < H):
            _need(state_out is None or state_out.data_ptr() != h0.data_ptr(), "a state in place needs contiguous rows that do not overlap")
            h0 = h0.contiguous()
    if lengths is not None:
        _need(lengths.device == dev and lengths.dtype == torch.int32 and tuple(lengths.shape) == (B,) and lengths.is_contiguous(),
              f"lengths must be contiguous int32 [{B}] on {dev}, got {lengths.dtype} {list(lengths.shape)} on {lengths.device}")
    wants_grad = torch.is_grad_enabled() and (pre.requires_grad or (h0 is not None and h0.requires_grad))
    if out is not None:
        _need(out.device == dev and out.dtype == pre.dtype and tuple(out.shape) == (B, T, H), f"out must be {pre.dtype} [{B}, {T}, {H}] on {dev}")
        _need((H <= 1 or out.stride(2) == 1) and _apart(out, H), "frames of out must be contiguous and not overlap")
        _need(not out.numel() or out.data_ptr() != pre.data_ptr(), "out must not be pre's memory")
    if state_out is not None:
        _need(state_out.device == dev, f"state_out must be on {dev}")
        _rows(state_out, B, H, "state_out")
        _need(h0 is None or state_out.data_ptr() != h0.data_ptr() or (h0.dim() == 2 and (B <= 1 or h0.stride(0) == state_out.stride(0))),
              "a state in place is h0 itself, one row per sequence")
    if wants_grad:
        _need(out is None and state_out is None, "out and state_out are for calls without gradients")
    with torch.cuda.device(dev):
        if wants_grad:
            h, last = _GatedScan.apply(pre, h0, lengths, bool(reverse))
            lib.guard_leaves(h.grad_fn)
            return h, last
        h, last, _ = _forward(pre, h0, lengths, reverse, out, state_out, False)
    return h, last
