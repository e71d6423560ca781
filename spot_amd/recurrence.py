"""Gated linear recurrence over sequences of any length on the GPU: the minGRU cell (reference model/min_gru.py:76-92) for whole
videos, frame streams and ragged batches, differentiable (stes_gated_scan_fwd / _bwd in include/stes.h).

    h, last = gated_scan(pre)                                    # [B, T, 2H] -> [B, T, H], fp32 [B, H]
    h, last = gated_scan(pre, h0=last)                           # the next frames of the same sequences
    gated_scan(pre, h0=state, state_out=state)                   # the same, the state updated in place
"""
from __future__ import annotations

import functools
import threading

import torch

from . import lib

_ELEMENT = {torch.bfloat16: 0, torch.float32: 1}


def _refuse(text):
    raise lib.StesError("gated_scan: " + text)


@functools.lru_cache(maxsize=256)
def _ws_bytes(B, T, H):
    return lib.lib().stes_gated_scan_ws_bytes(B, T, H)


class _Workspaces:
    """The two workspaces that the calls on one stream take in turn: a call finds its own zero and leaves the one of the call before
    zero, so none needs a launch that clears.  A call's launch happens under the lock: what is clean follows the stream's order."""

    def __init__(self):
        self.lock, self.pair, self.turn, self.dirty = threading.Lock(), None, 0, [0, 0]


_KEPT_BYTES = 16 << 20              # larger workspaces are not kept: clearing them is a small part of such calls (2 % of the data)
_KEPT_STREAMS = 64
_kept = {}                          # (device, stream) -> _Workspaces


def _call(entry, fields, dims, dev):
    """One call of the library with the workspace that it needs: `fields` are the arguments in front of it, `dims` those behind.  A
    captured call gets a workspace of its own, cleared in the graph: a graph may be replayed on any stream, next to others."""
    n = 0 if dims[1] <= lib.SCAN_BLOCK else _ws_bytes(*dims[:3])
    if not n:
        lib.call(entry, lib.pack_scan(*fields, 0, 0, 0, 0, 0, *dims))
        return
    if n > _KEPT_BYTES or torch.cuda.is_current_stream_capturing():
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        lib.call(entry, lib.pack_scan(*fields, ws.data_ptr(), n, 0, 0, 0, *dims))
        return
    key = (dev.index, lib.stream())
    k = _kept.get(key)
    if k is None:
        if len(_kept) >= _KEPT_STREAMS:
            _kept.pop(next(iter(_kept)), None)                 # (its memory goes back in its stream's order)
        k = _kept.setdefault(key, _Workspaces())
    with k.lock:
        if k.pair is None or k.pair[0].numel() < n:
            k.pair, k.turn, k.dirty = [torch.zeros(n, dtype=torch.uint8, device=dev) for _ in range(2)], 0, [0, 0]
        i, j = k.turn, 1 - k.turn
        try:
            lib.call(entry, lib.pack_scan(*fields, k.pair[i].data_ptr(), n, 1, k.pair[j].data_ptr() if k.dirty[j] else 0, k.dirty[j], *dims))
        except Exception:
            k.pair = None
            raise
        k.dirty[i], k.dirty[j], k.turn = n, 0, j


def _at(t):
    return 0 if t is None else t.data_ptr()


def _row_stride(t, B, H, name):
    """Stride between the rows of a float32 [B, H] tensor whose rows are contiguous and apart."""
    if t.dtype != torch.float32 or t.shape != (B, H):
        _refuse(f"{name} must be float32 [{B}, {H}], got {t.dtype} {list(t.shape)}")
    if (H > 1 and t.stride(1) != 1) or (B > 1 and t.stride(0) < H):
        _refuse(f"rows of {name} must be contiguous and not overlap")
    return t.stride(0) if B > 1 else max(H, 1)


def _strides(t, T, width):
    """(frame stride, sequence stride) of a [B, T, width] tensor; the frame stride of a single frame is immaterial."""
    bs, ld, _ = t.stride()
    return (ld if T > 1 else width), bs


def _apart(t, width):
    """Whether the rows of a [B, T, width] tensor with a contiguous last dimension are apart: frames within sequences or the reverse."""
    inner, outer = sorted((t.stride(i), t.shape[i]) if t.shape[i] > 1 else (0, 1) for i in (0, 1))
    if inner[1] > 1 and inner[0] < width:
        return False
    return outer[1] == 1 or outer[0] >= inner[0] * (inner[1] - 1) + width


def _forward(pre, h0, lengths, reverse, out, state_out, keep_states):
    B, T, W = pre.shape
    H, dev = W // 2, pre.device
    h = pre.new_empty(B, T, H) if out is None else out
    if state_out is None:
        last, bs_hl = torch.empty(B, H, dtype=torch.float32, device=dev), max(H, 1)
    else:
        last, bs_hl = state_out, _row_stride(state_out, B, H, "state_out")
    states = torch.empty(B, -(-T // lib.SCAN_BLOCK), H, dtype=torch.float32, device=dev) if keep_states else None
    if B and H:
        ld, bs = _strides(pre, T, W)
        ld_h, bs_h = (H, T * H) if out is None else _strides(h, T, H)
        _call("stes_gated_scan_fwd", (
            pre.data_ptr(), ld, bs, _at(h0), 0 if h0 is None or h0.dim() == 1 else _row_stride(h0, B, H, "h0"), _at(lengths),
            h.data_ptr(), ld_h, bs_h, last.data_ptr(), bs_hl, _at(states), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), (B, T, H, _ELEMENT[pre.dtype], reverse), dev)
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
        with lib.on_device(pre.device):
            return _backward(pre, lengths, states, ctx.reverse, ctx.h0_dim, dh, dlast)


def _backward(pre, lengths, states, reverse, h0_dim, dh, dlast):
    B, T, W = pre.shape
    H, dev = W // 2, pre.device
    dpre = torch.empty(B, T, W, dtype=pre.dtype, device=dev)
    dh0 = torch.empty(B, H, dtype=torch.float32, device=dev) if h0_dim else None
    total = torch.empty(H, dtype=torch.float32, device=dev) if h0_dim == 1 else None
    if H and (B or total is not None):
        ld, bs = _strides(pre, T, W)
        ld_dh = bs_dh = 0
        if dh is not None:
            if not dh.is_contiguous() and ((H > 1 and dh.stride(2) != 1) or (T > 1 and dh.stride(1) < H)):
                dh = dh.contiguous()                        # a gradient that was expanded or transposed
            ld_dh, bs_dh = _strides(dh, T, H)
        if dlast is not None:
            dlast = dlast.contiguous()
        _call("stes_gated_scan_bwd", (
            pre.data_ptr(), ld, bs, 0, 0, _at(lengths), 0, 0, 0, 0, 0, states.data_ptr(), _at(dh), ld_dh, bs_dh, _at(dlast), H,
            dpre.data_ptr(), W, T * W, _at(dh0), _at(total)), (B, T, H, _ELEMENT[pre.dtype], reverse), dev)
    return dpre, (total if h0_dim == 1 else dh0), None, None


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

    Differentiable (once) in pre and h0, from h and from the final states.  T = 0 and T = 1 are calls like any other."""
    if not isinstance(pre, torch.Tensor) or not pre.is_cuda or pre.dim() != 3 or pre.dtype not in _ELEMENT:
        _refuse("pre must be a bfloat16 or float32 tensor [B, T, 2H] on the GPU")
    B, T, W = pre.shape
    H, dev = W // 2, pre.device
    if W % 2:
        _refuse(f"the last dimension of pre holds gates and candidates and is even, got {W}")
    if not pre.is_contiguous() and ((W > 1 and pre.stride(2) != 1) or (T > 1 and pre.stride(1) < W)):
        _refuse("frames of pre must be contiguous and not overlap")
    if h0 is not None:
        if h0.device != dev or h0.dtype != torch.float32 or h0.shape not in ((B, H), (H,)):
            _refuse(f"h0 must be float32 [{B}, {H}] or [{H}] on {dev}, got {h0.dtype} {list(h0.shape)} on {h0.device}")
        if not h0.is_contiguous() and ((H > 1 and h0.stride(-1) != 1) or (h0.dim() == 2 and B > 1 and h0.stride(0) < H)):
            if state_out is not None and state_out.data_ptr() == h0.data_ptr():
                _refuse("a state in place needs contiguous rows that do not overlap")
            h0 = h0.contiguous()
    if lengths is not None and (lengths.device != dev or lengths.dtype != torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous()):
        _refuse(f"lengths must be contiguous int32 [{B}] on {dev}, got {lengths.dtype} {list(lengths.shape)} on {lengths.device}")
    wants_grad = torch.is_grad_enabled() and (pre.requires_grad or (h0 is not None and h0.requires_grad))
    if out is not None:
        if wants_grad:
            _refuse("out and state_out are for calls without gradients")
        if out.device != dev or out.dtype != pre.dtype or out.shape != (B, T, H) or (out.requires_grad and torch.is_grad_enabled()):
            _refuse(f"out must be {pre.dtype} [{B}, {T}, {H}] on {dev}, without gradients")
        if (H > 1 and out.stride(2) != 1) or not _apart(out, H):
            _refuse("frames of out must be contiguous and not overlap")
    if state_out is not None:
        if wants_grad:
            _refuse("out and state_out are for calls without gradients")
        if state_out.device != dev or (state_out.requires_grad and torch.is_grad_enabled()):
            _refuse(f"state_out must be on {dev}, without gradients")
        stride = _row_stride(state_out, B, H, "state_out")
        if h0 is not None and state_out.data_ptr() == h0.data_ptr() and B > 1 and (h0.dim() == 1 or h0.stride(0) != stride):
            _refuse("a state in place is h0 itself, one row per sequence")
    with lib.on_device(dev):
        if wants_grad:
            h, last = _GatedScan.apply(pre, h0, lengths, bool(reverse))
            lib.guard_leaves(h.grad_fn)
        else:
            h, last, _ = _forward(pre, h0, lengths, bool(reverse), out, state_out, False)
            lib.written(out, state_out)
    return h, last
