"""Gated linear recurrence over sequences of any length on the GPU: the minGRU cell (reference model/min_gru.py:76-92) for whole
videos, frame streams and ragged batches, differentiable (stes_gated_scan_fwd / _bwd in include/stes.h).

    h, last = gated_scan(pre)                                    # [B, T, 2H] -> [B, T, H], fp32 [B, H]
    h, last = gated_scan(pre, h0=last)                           # the next frames of the same sequences
    gated_scan(pre, h0=state, state_out=state)                   # the same, the state updated in place
"""
from __future__ import annotations

import torch

from . import lib


def gated_scan(pre, h0=None, lengths=None, reverse=False, out=None, state_out=None):
    """h_t = (1 - z_t) h_{t-1} + z_t c_t with z = sigmoid(pre[..., :H]) and c = pre[..., H:], along the frames of every sequence.

    pre      [B, T, 2H] bfloat16 or float32 on the GPU; the last dimension contiguous, any strides between frames and sequences
    h0       initial states: float32 [B, H], float32 [H] (one for the whole batch) or None (zeros)
    lengths  int32 [B] on the same device (values are clamped to [0, T]) or None: frames from a sequence's length on are not looked at,
             their h (and their gradients) are zero
    reverse  from a sequence's last frame to its first
    out, state_out (without gradients only): where h [B, T, H] and the final states float32 [B, H] go; state_out may be h0, apart
             from that they share no memory with one another or with what the call reads (columns of one buffer do not)
    -> h [B, T, H] in pre's type and the states after the last step, float32 [B, H] (h0 where a sequence is empty)

    A frame whose gates and candidates hold the type's lowest value leaves the states as they are; an infinite state stays infinite.

    Differentiable (once) in pre and h0, from h and from the final states; not to be traced.  T = 0 and T = 1 are calls like any other."""
    if not isinstance(pre, torch.Tensor):
        raise lib.StesError(f"gated_scan: pre must be a tensor, got {type(pre).__name__}")
    return lib.native_call("gated_scan_kernel", lib.native().gated_scan, pre, h0, lengths, reverse, out, state_out)
