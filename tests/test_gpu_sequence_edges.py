"""The gated scan and the distillation loss at the ends of their types and of their interfaces, on the GPU, against the 64-bit
restatements (oracle/sequence_oracle.py): tolerances are the oracle's bounds plus half a step of the type that a result is stored in."""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO
from test_gpu_sequence import _check, _differentiable_calls, _kl_compare, _kl_inputs, _np, _run_scan, _scan_inputs

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _against_the_oracle(pre, start, lengths, dh, dlast, reverse):
    with np.errstate(all="ignore"):
        ref = SO.gated_scan(_np(pre), _np(start), _np(lengths), reverse, _np(dh), _np(dlast), need_grad=True)
        got = _run_scan_any(pre, start, lengths, dh, dlast, reverse)
        for name, t in zip(("h", "last", "dpre", "dh0"), got):
            _check(t, ref[name], ref[name + "_err"], name)
    return ref, got


def _run_scan_any(pre, start, lengths, dh, dlast, reverse):
    """_run_scan without its comparison of two calls by torch.equal, which NaN fails."""
    from spot_amd.recurrence import gated_scan
    p, s = pre.cuda().requires_grad_(), start.cuda().requires_grad_()
    h, last = gated_scan(p, h0=s, lengths=None if lengths is None else lengths.cuda(), reverse=reverse)
    return (h, last) + torch.autograd.grad((h, last), (p, s), (dh.cuda(), dlast.cuda()))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,T,H", [(F32, 1, 5), (F32, 5, 8), (BF, 8, 16), (BF, 64, 72), (F32, 300, 24), (BF, 1000, 40)])
def test_gated_scan_frames_masked_with_the_lowest_value(dtype, T, H, reverse):
    """Frames whose gates and candidates hold the type's lowest value leave the state as it is: sigmoid is 0 there, and 0 times the
    lowest value is 0.  Their gates' and candidates' gradients are exactly zero."""
    pre, start, lengths, dh, dlast = _scan_inputs(3, T, H, dtype, True, "rows", seed=T + H)
    masked = torch.rand(3, T, generator=torch.Generator().manual_seed(T)) < 0.6
    masked[2] |= T == 1
    pre[masked] = torch.finfo(dtype).min
    _, got = _against_the_oracle(pre, start, lengths, dh, dlast, reverse)
    assert not bool(got[2].cpu()[masked].any())
    pre[:] = torch.finfo(dtype).min
    h, last, dpre, _ = _run_scan(pre, start, None, dh, dlast, reverse)
    assert torch.equal(last.cpu(), start) and torch.equal(h.cpu(), start.to(dtype)[:, None].expand(3, T, H)) and not bool(dpre.any())


@pytest.mark.parametrize("dtype,T,H", [(F32, 4, 6), (BF, 8, 16), (BF, 200, 16), (F32, 200, 9), (F32, 700, 12)])
def test_gated_scan_gradients_of_saturated_gates(dtype, T, H):
    """Gates at and beyond the end of the type's range, the gradients to the oracle's bound: exactly zero at the gates, and at the
    candidates of closed ones."""
    pre, start, _, dh, dlast = _scan_inputs(2, T, H, dtype, False, "rows", seed=8)
    v = torch.tensor([INF, -INF, torch.finfo(dtype).max, torch.finfo(dtype).min, 0.0, 30.0, -30.0, 1.0])
    pick = torch.randint(0, 8, (2, T, H), generator=torch.Generator().manual_seed(1))
    pre[..., :H] = v[pick].to(dtype)
    _, got = _against_the_oracle(pre, start, None, dh, dlast, False)
    dgate, dcand = got[2].cpu()[..., :H], got[2].cpu()[..., H:]
    assert float(dgate[pick < 4].abs().max()) <= 1e-37 and not bool(dcand[(pick == 1) | (pick == 3)].any())
    assert float(dgate[pick == 7].abs().max()) > 0.01 and float(dcand[pick == 0].abs().max()) > 0.5


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,T,H", [(F32, 6, 16), (BF, 64, 64), (F32, 250, 20), (BF, 600, 64), (F32, 3000, 12)])
def test_gated_scan_infinite_states_stay_infinite(dtype, T, H, reverse):
    """Infinite initial states, candidates and gradients: what comes behind one is infinite, NaN only where two of other signs meet,
    whatever the length and however the time axis is cut."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, dh, dlast = _scan_inputs(3, T, H, dtype, False, "rows", seed=T, gate=(0.0, 1.5))
    start[0, 0], start[1, 1], start[2, 2] = INF, -INF, NAN
    pre[0, T // 2, H + 3], pre[1, T // 3, H + 4], pre[2, T - 1, H + 5] = INF, -INF, INF
    pre[0, T // 3, H + 6], pre[0, T // 2, H + 6] = INF, -INF
    dh[1, T // 2, 7], dh[2, T // 2, 8], dlast[0, 9] = INF, -INF, INF
    ref, got = _against_the_oracle(pre, start, None, dh, dlast, reverse)
    assert np.isinf(ref["last"][0, 0]) and np.isinf(ref["dh0"][1, 7]) and np.isinf(ref["dh0"][0, 9])
    state, parts, p = start.cuda(), [], pre.cuda()
    for lo, hi in ((0, T // 2), (T // 2, T)) if not reverse else ((T // 2, T), (0, T // 2)):
        h, state = gated_scan(p[:, lo:hi], state, reverse=reverse)
        parts.append(h)
    both = torch.cat(parts[::-1] if reverse else parts, 1)
    for a, b in ((both, got[0]), (state, got[1])):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf()) and torch.equal(a[a.isinf()], b[b.isinf()])


def test_tangents_are_refused_in_backward_passes_and_in_results():
    """A tangent that arrives with the upstream gradient, or that a result to be written carries, would be lost without a word."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad
    from spot_amd.recurrence import gated_scan
    ad = torch.autograd.forward_ad
    for leaf, f in _differentiable_calls():
        y = f(leaf)
        with ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
        torch.autograd.grad(y, leaf)
    p = torch.randn(2, 3, 8, device="cuda", requires_grad=True)
    h, last = gated_scan(p)
    with ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(last, p, ad.make_dual(torch.ones_like(last), torch.ones_like(last)))
        dual = lambda *s: ad.make_dual(torch.zeros(*s, device="cuda"), torch.ones(*s, device="cuda"))  # noqa: E731
        for kw in (dict(out=dual(2, 3, 4)), dict(state_out=dual(2, 4))):
            with pytest.raises(lib.StesError, match="forward-mode"):
                gated_scan(p.detach(), **kw)
        with pytest.raises(lib.StesError, match="forward-mode"):
            topk_distill_grad(torch.zeros(4, 7, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, 2, device="cuda"), out=dual(4, 7))


def test_tracing_refuses_forward_and_backward_passes():
    from torch.fx.experimental.proxy_tensor import make_fx
    from spot_amd import lib
    for leaf, f in _differentiable_calls():
        want = f(leaf)
        with pytest.raises(lib.StesError, match="trace"):
            make_fx(f)(leaf.detach())
        with pytest.raises(lib.StesError, match="trace"):
            torch.jit.trace(f, (leaf.detach(),), check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(lambda u: torch.autograd.grad(want, leaf, u, retain_graph=True)[0])(torch.ones_like(want))
        torch.autograd.grad(want, leaf)
        from torch.utils.flop_counter import FlopCounterMode
        with FlopCounterMode(display=False):                # a mode that only looks on
            assert torch.equal(f(leaf), want)


@pytest.mark.parametrize("B", [34, 100, 192])
@pytest.mark.parametrize("T", [2, 5, 300])
def test_gated_scan_in_columns_of_a_time_major_buffer(B, T):
    """[T][B][3H], frames outermost: pre in the first 2H columns, the states written beside them; one column more is refused."""
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    H = 8
    pre, start, _, _, _ = _scan_inputs(B, T, H, F32, False, "rows", seed=B + T)
    want = gated_scan(pre.cuda(), start.cuda())
    buf = torch.full((T, B, 3 * H), NAN, device="cuda")
    view = buf.transpose(0, 1)
    view[..., :2 * H] = pre.cuda()
    h, last = gated_scan(view[..., :2 * H], start.cuda(), out=view[..., 2 * H:])
    assert torch.equal(h, want[0]) and torch.equal(last, want[1]) and torch.equal(view[..., :2 * H], pre.cuda())
    for out in (view[..., 2 * H - 1:3 * H - 1], view[..., :H]):
        with pytest.raises(lib.StesError):
            gated_scan(view[..., :2 * H], start.cuda(), out=out)


def test_capture_accepts_leaves_of_its_own_stream_and_refuses_others():
    """A leaf that an eager graph holds is refused in a capture for the stream that graph ran on, whoever made the graph: one that ran on the
    capture's own stream does no harm, one that torch's own functions made does."""
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    for leaf, f in _differentiable_calls():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            alive = f(leaf)
            want, = torch.autograd.grad(alive, leaf, retain_graph=True)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            g, = torch.autograd.grad(f(leaf), leaf)
        for _ in range(3):
            g.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(g, want)
        del alive
    p = torch.randn(2, 4, 16, device="cuda", requires_grad=True)
    alive = (p * 2).sum()                                   # on the default stream
    torch.cuda.synchronize()
    with pytest.raises(lib.StesError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.ones(4, device="cuda").mul_(2)
            gated_scan(p)
    del alive


@pytest.mark.parametrize("V", [7, 300, 1000, 20000, 70000])
def test_distill_statistics_are_the_maximum_and_the_sum(V):
    """The contract of the C interface: stats hold a row's maximum and sum exp((logits - max) / tau), and the backward pass takes what the
    caller gives."""
    import ctypes as C
    from spot_amd import lib
    M, k, tau = 6, 3, 2.0
    s, idx, val, _ = _kl_inputs(M, V, k, F32, V)
    x, i, v = s.cuda(), idx.cuda(), val.cuda()
    stats, loss, d = torch.full((M, 2), NAN, device="cuda"), torch.zeros(1, device="cuda"), torch.full((M, V), NAN, device="cuda")
    n = lib.lib().stes_distill_ws_floats(M, V, k, 0)
    ws = torch.zeros(max(n, 1), device="cuda")
    base = dict(logits=lib.ptr(x), ld=V, f32=1, idx=lib.ptr(i), ld_idx=k, idx_i64=1, val=lib.ptr(v), ld_val=k, val_f32=1, M=M, V=V, k=k, temperature=tau, denom=3.0,
                grad_scale=1.0)

    def args(**kw):
        a = lib.DistillArgs()
        for name, value in {**base, **kw}.items():
            setattr(a, name, value)
        return a
    a = args(loss=lib.ptr(loss), stats=lib.ptr(stats), ws=lib.ptr(ws), ws_floats=n)
    lib.check(lib.lib().stes_distill(C.byref(a), lib.stream()), "stes_distill")
    top = _np(s).max(1)
    y = (_np(s) - top[:, None]) / tau
    total = np.exp(y).sum(1)
    _check(stats[:, 0], top, 0 * top, "maximum")
    # exp2 of a rounded argument (3 u |y|) good to 2 u, and fewer than V / 4 + 16 roundings of the sum
    _check(stats[:, 1], total, SO.U * ((np.exp(y) * (4 * np.abs(y) + 2)).sum(1) + (V / 4 + 16) * total), "sum")
    given = torch.tensor(np.stack([top, total], 1), dtype=F32, device="cuda")
    a = args(stats=lib.ptr(given), dlogits=lib.ptr(d), ld_d=V, d_f32=1)
    lib.check(lib.lib().stes_distill_bwd(C.byref(a), lib.stream()), "stes_distill_bwd")
    ref = SO.topk_distill(_np(s), _np(idx), _np(val), tau, None, 3.0)
    _check(d, ref["dlogits"], ref["dlogits_err"], "dlogits")


def test_streams_from_outside_keep_no_workspaces():
    """A stream that torch did not make may be destroyed and its handle given out again: nothing is kept for it."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(2, 900, 96, BF, False, "rows", seed=8)
    s, idx, val, _ = _kl_inputs(5000, 40, 4, F32, 1)
    p, h0, c = pre.cuda().requires_grad_(), start.cuda(), (s.cuda(), idx.cuda(), val.cuda())

    def work():
        h, last = gated_scan(p, h0)
        return (h.detach(), last.detach(), torch.autograd.grad(h, p, torch.ones_like(h))[0]) + topk_distill_grad(*c)
    want = work()
    mine = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = lib.native().kept_streams()
    got = []
    with torch.cuda.stream(torch.cuda.ExternalStream(mine.cuda_stream)):
        for _ in range(3):
            got.append(work())
    torch.cuda.synchronize()
    assert lib.native().kept_streams() == before
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.parametrize("V", [6, 300, 700, 9000, 80000])
@pytest.mark.parametrize("dtype,tau", [(F32, 1.0), (BF, 1.0), (F32, 0.5), (BF, 4.0)])
def test_distill_listed_classes_at_the_lowest_value(V, dtype, tau):
    """A class that the teacher lists and the student masks with the type's lowest value: the divergence is of the order of 3e38 and finite, in
    one row and where several rows' sum alone passes the range of fp32."""
    M = 9
    s, idx, val, w = _kl_inputs(M, V, 2, dtype, V + 1, False, True)
    for m in (1, 2, 3, 4, 8):
        s[m, idx[m, m % 2]] = torch.finfo(dtype).min
    ref = _kl_compare(s, idx, val, None, tau, denom=100.0)
    assert np.isfinite(ref["loss"]) and 1e36 < ref["loss"] < 1e38
    _kl_compare(s, idx, val, 4 * w, tau, denom=1000.0)


def test_threads_on_one_stream_while_allocations_are_recorded():
    """Recording an allocation takes the interpreter's lock: a thread that waits for the workspaces that another one allocates must not keep it."""
    import threading
    from spot_amd.recurrence import gated_scan
    torch.cuda.synchronize()
    shared, done = torch.cuda.Stream(), []

    def work(k):
        with torch.cuda.stream(shared):
            for i in range(1, 16):                          # (growing: every call allocates its workspaces anew)
                p = torch.zeros(1, 300, 32 * (16 * k + i), device="cuda", requires_grad=True)
                h, _ = gated_scan(p)
                g, = torch.autograd.grad(h, p, torch.ones_like(h))
                done.append(bool(g.any()))
    torch.cuda.memory._record_memory_history("all", stacks="python", max_entries=1000)
    try:
        threads = [threading.Thread(target=work, args=(k,), daemon=True) for k in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(30)
    finally:
        torch.cuda.memory._record_memory_history(None)
    assert len(done) == 45


@pytest.mark.parametrize("T", [0, 5, 300])
def test_gated_scan_of_no_sequences_has_a_zero_gradient_of_the_shared_state(T):
    from spot_amd.recurrence import gated_scan
    p, s = torch.zeros(0, T, 16, device="cuda", requires_grad=True), torch.randn(8, device="cuda", requires_grad=True)
    h, last = gated_scan(p, s)
    g = torch.autograd.grad((h, last), (p, s), (torch.ones_like(h), torch.ones_like(last)))
    assert g[0].shape == p.shape and g[1].shape == (8,) and not bool(g[1].any())


def test_captures_on_two_streams_share_a_leaf():
    """The outputs of one capture hold a leaf whose gradient's node was made on that capture's stream: another capture's forward pass takes it."""
    for leaf, f in _differentiable_calls():
        want = f(leaf).detach().clone()
        torch.cuda.synchronize()
        kept = []
        for _ in range(2):
            gr, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(gr, stream=side):
                kept.append((gr, f(leaf), side))
        for gr, y, _ in kept:
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_saved_tensors_may_come_back_with_other_strides_and_are_refused_as_others():
    """What hooks give back for a saved tensor: the same values in another layout do, another size or type is refused."""
    hooks = torch.autograd.graph.saved_tensors_hooks

    def apart(t):                                           # every element on its own, the last dimension outermost
        if t.dim() < 2 or not t.numel():
            return torch.stack([t, t], -1)[..., 0]
        return t.movedim(-1, 0).contiguous().movedim(0, -1)
    for leaf, f in _differentiable_calls():
        want, = torch.autograd.grad(f(leaf), leaf)
        with hooks(lambda t: t.clone(), apart):
            y = f(leaf)
        assert torch.equal(torch.autograd.grad(y, leaf)[0], want)
        for change in (lambda t: t[..., :-1], lambda t: t.double(), lambda t: t.cpu(), lambda t: t[None]):
            with hooks(lambda t: t, lambda t, change=change: change(t) if t.shape == leaf.shape and t.data_ptr() == leaf.data_ptr() else t):
                y = f(leaf)
            with pytest.raises(RuntimeError, match="came back as"):
                torch.autograd.grad(y, leaf)


def test_lazily_negated_and_lazily_zero_tensors():
    """Tensors whose memory does not hold their values (torch's negative views, its zero tensors without memory) are read as their values;
    results are not written through them."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    from spot_amd.recurrence import gated_scan
    neg = torch._neg_view
    pre, start, _, dh, dlast = _scan_inputs(2, 40, 8, F32, False, "rows", seed=3)
    p, s, d, dl = pre.cuda().requires_grad_(), start.cuda().requires_grad_(), dh.cuda(), dlast.cuda()
    zero = torch._efficientzerotensor(2, 8, device="cuda")

    def scan(a, b, u, v):
        y = gated_scan(a, b)
        return y + torch.autograd.grad(y, (p, s), (u, v))
    want = scan(p, s, d, dl)
    for got in (scan(neg(-p), s, d, dl), scan(p, neg(-s), d, dl), scan(p, s, neg(-d), neg(-dl))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    z = torch.zeros(2, 8, device="cuda")
    for a, b in zip(scan(p, s, d, zero), scan(p, s, d, z)):
        assert torch.equal(a, b)
    assert torch.equal(gated_scan(p.detach(), zero)[0], gated_scan(p.detach(), z)[0])
    for kw in (dict(out=neg(torch.zeros(2, 40, 8, device="cuda"))), dict(state_out=neg(z.clone())), dict(state_out=torch._efficientzerotensor(2, 8, device="cuda"))):
        with pytest.raises(lib.StesError):
            gated_scan(p.detach(), **kw)
    x, idx, val, w = _kl_inputs(9, 30, 4, F32, 2, False, True)
    x, idx, val, w, up = x.cuda().requires_grad_(), idx.cuda(), val.cuda(), w.cuda(), torch.tensor(0.5, device="cuda")

    def kl(a, v, wt, u):
        y = topk_distill_loss(a, idx, v, 2.0, wt)
        return (y, torch.autograd.grad(y, x, u)[0]) + topk_distill_grad(a, idx, v, 2.0, wt)
    want = kl(x, val, w, up)
    for got in (kl(neg(-x), val, w, up), kl(x, neg(-val), w, up), kl(x, val, neg(-w), up), kl(x, val, w, neg(-up))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = kl(x, val, torch._efficientzerotensor(9, device="cuda"), torch._efficientzerotensor((), device="cuda"))
    assert float(none[0]) == 0 and not bool(none[1].any()) and float(none[2]) == 0 and not bool(none[3].any())
    g, = torch.autograd.grad(topk_distill_loss(x, idx, val), x, torch._efficientzerotensor((), device="cuda"))
    assert not bool(g.any())
    with pytest.raises(lib.StesError):
        topk_distill_grad(x.detach(), idx, val, out=neg(torch.zeros(9, 30, device="cuda")))
