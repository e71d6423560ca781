"""Gated scan and top-logits distillation on the GPU against their 64-bit restatements (oracle/sequence_oracle.py): the tolerances are
the running error bounds that the oracle derives from the inputs, plus half a step of the type that a result is stored in."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from oracle import sequence_oracle as SO

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _check(got, ref, err, what):
    """Elementwise |got - ref| <= err + half a step of got's type at the value; infinities and NaN in the same places."""
    half = torch.finfo(got.dtype).eps / 2
    got, ref, err = got.detach().double().cpu().numpy(), np.asarray(ref), np.asarray(err)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = np.isfinite(ref)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref), err_msg=what)
    np.testing.assert_array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)], err_msg=what)
    off = np.abs(got - ref)[fine] - (err + half * (np.abs(ref) + err) + 1e-37)[fine]
    assert off.size == 0 or off.max() <= 0, (what, float(off.max()), int((off > 0).sum()), off.size)


# ------------------------------------------------------------------------------------------------------------- scan
def _scan_inputs(B, T, H, dtype, ragged, h0, seed, gate=(-1.5, 2.0)):
    g = torch.Generator().manual_seed(seed)
    pre = torch.randn(B, T, 2 * H, generator=g)
    pre[..., :H] = pre[..., :H] * gate[1] + gate[0]
    pre = pre.to(dtype)
    start = {"rows": torch.randn(B, H, generator=g), "shared": torch.randn(H, generator=g), "none": None}[h0]
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        lengths[0] = 0
        lengths[-1] = T
    return pre, start, lengths, torch.randn(B, T, H, generator=g).to(dtype), torch.randn(B, H, generator=g)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _run_scan(pre, start, lengths, dh, dlast, reverse):
    from spot_amd.recurrence import gated_scan
    p = pre.cuda().requires_grad_()
    s = None if start is None else start.cuda().requires_grad_()
    n = None if lengths is None else lengths.cuda()
    h, last = gated_scan(p, h0=s, lengths=n, reverse=reverse)
    g = torch.autograd.grad((h, last), (p,) if s is None else (p, s), (dh.cuda(), dlast.cuda()))
    with torch.no_grad():
        h2, last2 = gated_scan(p, h0=s, lengths=n, reverse=reverse)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    return h, last, g[0], (g[1] if s is not None else None)


def _compare_scan(pre, start, lengths, dh, dlast, reverse, got):
    ref = SO.gated_scan(_np(pre), _np(start), _np(lengths), reverse, _np(dh), _np(dlast), need_grad=True)
    h, last, dpre, dh0 = got
    _check(h, ref["h"], ref["h_err"], "h")
    _check(last, ref["last"], ref["last_err"], "last")
    _check(dpre, ref["dpre"], ref["dpre_err"], "dpre")
    if start is not None:
        r, e = ref["dh0"], ref["dh0_err"]
        if start.dim() == 1:
            r, e = r.sum(0), e.sum(0) + r.shape[0] * SO.U * np.abs(r).sum(0)
        _check(dh0, r, e, "dh0")


SCAN_CASES = [  # B, T, H, dtype, ragged, reverse, h0
    (1, 1, 1, F32, False, False, "rows"), (3, 1, 768, BF, False, False, "rows"), (2, 2, 5, BF, True, True, "shared"),
    (70, 3, 16, BF, False, False, "none"), (5, 7, 24, F32, True, False, "rows"), (4, 8, 64, BF, False, True, "rows"),
    (4, 9, 64, BF, True, False, "shared"), (2, 31, 33, BF, False, False, "rows"), (3, 64, 768, BF, False, False, "shared"),
    (3, 127, 40, F32, True, True, "rows"), (2, 128, 136, BF, False, False, "rows"), (2, 129, 128, BF, True, True, "none"),
    (2, 129, 7, F32, False, False, "rows"), (6, 255, 12, F32, True, False, "rows"), (3, 256, 68, BF, True, False, "rows"),
    (2, 257, 260, F32, False, True, "shared"), (5, 700, 200, BF, True, False, "rows"), (1, 1000, 264, BF, False, False, "rows"),
    (1, 1025, 130, F32, False, True, "rows"), (2, 3001, 9, BF, True, True, "shared"), (1, 9000, 8, F32, False, False, "rows"),
    (1, 20000, 3, BF, False, True, "rows"), (40, 130, 64, BF, True, False, "shared"), (700, 2, 70, F32, True, False, "shared"),
]


@pytest.mark.parametrize("B,T,H,dtype,ragged,reverse,h0", SCAN_CASES)
def test_gated_scan_and_gradients(B, T, H, dtype, ragged, reverse, h0):
    x = _scan_inputs(B, T, H, dtype, ragged, h0, seed=B * 1000 + T)
    _compare_scan(*x, reverse, _run_scan(*x, reverse))


@pytest.mark.parametrize("dtype,T", [(BF, 5), (BF, 300), (F32, 300), (F32, 1)])
def test_gated_scan_gates_nearly_closed_keep_a_long_memory(dtype, T):
    """Gates of 1e-4 on average: a state is a sum over the whole sequence, carried over every tile border."""
    x = _scan_inputs(2, T, 72, dtype, False, "rows", seed=5, gate=(-9.0, 1.0))
    _compare_scan(*x, False, _run_scan(*x, False))


@pytest.mark.parametrize("dtype,H", [(BF, 16), (F32, 16), (BF, 9)])
def test_gated_scan_saturated_gates(dtype, H):
    """Gates at and beyond the end of the type's range: z = 0 keeps the state, z = 1 replaces it, gradients of both are zero."""
    pre, start, _, dh, dlast = _scan_inputs(2, 200, H, dtype, False, "rows", seed=8)
    v = torch.tensor([100.0, -100.0, INF, -INF, torch.finfo(dtype).max, torch.finfo(dtype).min, 0.0, 30.0])
    pre[..., :H] = v[torch.randint(0, 8, (2, 200, H), generator=torch.Generator().manual_seed(1))].to(dtype)
    p64 = _np(pre)
    with np.errstate(over="ignore"):
        p64[..., :H] = np.clip(p64[..., :H], -1e4, 1e4)             # (the oracle's bound needs a finite gate; sigmoid is 0 or 1 there alike)
    h, last, dpre, dh0 = _run_scan(pre, start, None, dh, dlast, False)
    ref = SO.gated_scan(p64, _np(start), None, False, _np(dh), _np(dlast), need_grad=True)
    # every |x| in the bound counts as at most 104 (a gate of exactly 0 or 1 has no error): states are sums of at most 200 terms
    bound = 200 * 116 * SO.U * (np.abs(p64[..., H:]).max() + np.abs(_np(start)).max())
    _check(h, ref["h"], np.full(ref["h"].shape, bound), "h")
    _check(last, ref["last"], np.full(ref["last"].shape, bound), "last")
    scale = np.abs(_np(dh)).max() * 200 + np.abs(_np(dlast)).max()
    worst = bound * scale + 400 * 116 * SO.U * scale * np.abs(p64[..., H:]).max() * 2
    _check(dpre, ref["dpre"], np.full(ref["dpre"].shape, worst), "dpre")
    _check(dh0, ref["dh0"], np.full(ref["dh0"].shape, worst), "dh0")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,T,H", [(BF, 6, 16), (BF, 300, 72), (F32, 300, 7)])
def test_gated_scan_padding_is_not_looked_at(dtype, T, H, reverse):
    """NaN and infinities behind a sequence's length reach neither the states nor the gradients; rows there are zero; a sequence of
    length 0 hands its initial state (and the gradient of its final one) through."""
    pre, start, _, dh, dlast = _scan_inputs(4, T, H, dtype, False, "rows", seed=T)
    lengths = torch.tensor([0, 1, T // 2, T], dtype=torch.int32)
    dirty, ddirty = pre.clone(), dh.clone()
    for b in range(4):
        dirty[b, lengths[b]:, :H] = torch.tensor([NAN, INF, -INF])[torch.arange(T - int(lengths[b])) % 3][:, None].to(dtype)
        dirty[b, lengths[b]:, H:] = NAN
        ddirty[b, lengths[b]:] = INF
    got = _run_scan(dirty, start, lengths, ddirty, dlast, reverse)
    clean = _run_scan(pre, start, lengths, dh, dlast, reverse)
    for a, b in zip(got, clean):
        assert torch.equal(a, b)
    _compare_scan(pre, start, lengths, dh, dlast, reverse, got)
    assert torch.equal(got[1][0].cpu(), start[0]) and torch.equal(got[3][0].cpu(), dlast[0])
    assert float(got[0][1, 1:].abs().max()) == 0 and float(got[2][1, 1:].abs().max()) == 0


def test_gated_scan_of_one_sequence_seen_several_times():
    """pre expanded over the batch (no memory of its own per sequence), from other states and over other lengths: gradients of the
    sequences add up in the one that is there."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, dh, dlast = _scan_inputs(3, 280, 20, F32, False, "rows", seed=6)
    n = torch.tensor([280, 3, 0], dtype=torch.int32)
    p, s = pre[:1].cuda().requires_grad_(), start.cuda().requires_grad_()
    h, last = gated_scan(p.expand(3, 280, 40), s, n.cuda())
    g = torch.autograd.grad((h, last), (p, s), (dh.cuda(), dlast.cuda()))
    ref = SO.gated_scan(_np(pre[:1]).repeat(3, 0), _np(start), _np(n), False, _np(dh), _np(dlast), need_grad=True)
    _check(h, ref["h"], ref["h_err"], "h")
    _check(last, ref["last"], ref["last_err"], "last")
    _check(g[0], ref["dpre"].sum(0, keepdims=True), ref["dpre_err"].sum(0, keepdims=True) + 4 * SO.U * np.abs(ref["dpre"]).sum(0, keepdims=True), "dpre")
    _check(g[1], ref["dh0"], ref["dh0_err"], "dh0")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H", [(1, 16), (7, 5), (300, 40)])
def test_gated_scan_in_columns_and_frames_of_one_buffer(T, H, dtype):
    """The output beside the input in one buffer, in its columns or behind it in time, and states beside one another: as with memory of
    their own; what would share memory is refused."""
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(3, T, H, dtype, False, "rows", seed=T)
    want = gated_scan(pre.cuda(), start.cuda())
    buf = torch.full((3, T, 3 * H), NAN, dtype=dtype, device="cuda")
    buf[..., :2 * H] = pre.cuda()
    st = torch.full((3, 2 * H), NAN, device="cuda")
    st[:, :H] = start.cuda()
    h, last = gated_scan(buf[..., :2 * H], st[:, :H], out=buf[..., 2 * H:], state_out=st[:, H:])
    assert torch.equal(h, want[0]) and torch.equal(last, want[1]) and torch.equal(buf[..., :2 * H], pre.cuda()) and torch.equal(st[:, :H], start.cuda())
    long = torch.full((3, 2 * T, 2 * H), NAN, dtype=dtype, device="cuda")
    long[:, :T] = pre.cuda()
    h, _ = gated_scan(long[:, :T], st[:, :H], out=long[:, T:, :H])
    assert torch.equal(h, want[0]) and torch.equal(long[:, :T], pre.cuda()) and bool(torch.isnan(long[:, T:, H:]).all())
    x = buf[..., :2 * H]
    for kw in (dict(out=x[..., :H]), dict(out=x[..., H:]), dict(out=buf[..., 2 * H - 1:3 * H - 1]), dict(out=long[:, T:, :H], pre=long[:, T:]),
               dict(state_out=st[:, 1:H + 1]), dict(h0=st[0, :H], state_out=st[:, :H])):
        with pytest.raises(lib.StesError):
            gated_scan(kw.pop("pre", x), kw.pop("h0", st[:, :H]), **kw)


def test_results_in_place_are_seen_by_autograd():
    """A graph that saved what a call then overwrites refuses its backward pass, as with torch's own functions; results that ask for
    gradients are refused."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad
    from spot_amd.recurrence import gated_scan
    pre, state = torch.zeros(2, 5, 8, device="cuda"), torch.ones(2, 4, device="cuda")
    out = torch.zeros(2, 5, 4, device="cuda")
    w = torch.ones(2, 4, device="cuda", requires_grad=True)
    y = (w * state).sum()
    gated_scan(pre, state, state_out=state)
    with pytest.raises(RuntimeError):
        y.backward()
    v = torch.ones(2, 5, 4, device="cuda", requires_grad=True)
    y = (v * out).sum()
    gated_scan(pre, state, out=out)
    with pytest.raises(RuntimeError):
        y.backward()
    s, i, t = torch.zeros(4, 7, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, 2, device="cuda")
    d, u = torch.zeros(4, 7, device="cuda"), torch.ones(4, 7, device="cuda", requires_grad=True)
    y = (u * d).sum()
    topk_distill_grad(s, i, t, out=d)
    with pytest.raises(RuntimeError):
        y.backward()
    for kw in (dict(out=v), dict(state_out=w)):
        with pytest.raises(lib.StesError):
            gated_scan(pre, **kw)
    with pytest.raises(lib.StesError):
        topk_distill_grad(s, i, t, out=u)
    with torch.inference_mode():
        a, b = torch.zeros(2, 5, 4, device="cuda"), torch.zeros(2, 4, device="cuda")
        gated_scan(pre, b, out=a, state_out=b)
        topk_distill_grad(s, i, t, out=torch.zeros(4, 7, device="cuda"))
    with torch.no_grad():
        gated_scan(pre, out=v)


@pytest.mark.parametrize("V", [7, 1000, 40000])
def test_distill_gradient_beside_the_logits(V):
    """The gradient in other columns of the logits' buffer; what would share memory, or has no single row stride, is refused."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad
    s, idx, val, w = _kl_inputs(4, V, 3, F32, V, False, True)
    c = (idx.cuda(), val.cuda(), 2.0, w.cuda())
    want = topk_distill_grad(s.cuda(), *c)
    buf = torch.full((4, 2 * V), NAN, device="cuda")
    buf[:, :V] = s.cuda()
    loss, d = topk_distill_grad(buf[:, :V], *c, out=buf[:, V:])
    assert torch.equal(loss, want[0]) and torch.equal(buf[:, V:], want[1]) and torch.equal(buf[:, :V], s.cuda())
    for out in (buf[:, :V], buf[:, V - 1:2 * V - 1], buf.view(torch.bfloat16)[:, :V]):
        with pytest.raises(lib.StesError):
            topk_distill_grad(buf[:, :V], *c, out=out)
    with pytest.raises(lib.StesError):
        topk_distill_grad(s.cuda().view(2, 2, V), idx.cuda().view(2, 2, 3), val.cuda().view(2, 2, 3), out=torch.zeros(2, 3, V, device="cuda")[:, :2])


def test_gated_scan_clamps_lengths():
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(3, 140, 8, BF, False, "rows", seed=0)
    n = torch.tensor([-5, 141, 1 << 30], dtype=torch.int32).cuda()
    h, last = gated_scan(pre.cuda(), start.cuda(), n)
    w, wl = gated_scan(pre.cuda(), start.cuda())
    assert torch.equal(h[1:], w[1:]) and torch.equal(last[1:], wl[1:]) and not bool(h[0].any()) and torch.equal(last[0].cpu(), start[0])


@pytest.mark.parametrize("dtype,H,off", [(BF, 64, 0), (BF, 64, 1), (BF, 60, 4), (F32, 24, 2), (F32, 24, 4), (BF, 11, 3)])
def test_gated_scan_strides_and_alignment(dtype, H, off):
    """Rows inside wider rows at any offset, sequences with gaps or in another order, gradients expanded from one row: the bits of the
    contiguous call."""
    from spot_amd.recurrence import gated_scan
    B, T = 3, 261
    pre, start, _, dh, _ = _scan_inputs(B, T, H, dtype, False, "rows", seed=H + off)
    wide = torch.full((T + 2, B + 1, 2 * H + 13), NAN, dtype=dtype).cuda()
    wide[:T, :B, off:off + 2 * H] = pre.transpose(0, 1).cuda()
    view = wide[:T, :B, off:off + 2 * H].transpose(0, 1)               # [B, T, 2H], frames outermost in memory
    wide0 = torch.full((B, H + 5), NAN).cuda()
    wide0[:, 1:H + 1] = start.cuda()
    both = torch.full((B, T, 2 * H + 3), 7.0, dtype=dtype).cuda()
    h, last = gated_scan(pre.cuda(), start.cuda())
    half = both[..., off:off + H]
    state = wide0[:, 1:H + 1]
    hv, lv = gated_scan(view, state, out=half, state_out=state)         # the state in place, rows with gaps
    _check(hv, _np(h), 0 * _np(h) + 1e-4, "h")                          # (another alignment may take another split of the time axis)
    ref = SO.gated_scan(_np(pre), _np(start))
    _check(hv, ref["h"], ref["h_err"], "h")
    _check(lv, ref["last"], ref["last_err"], "last")
    assert hv.data_ptr() == half.data_ptr() and lv.data_ptr() == state.data_ptr() and bool(wide0[:, 0].isnan().all()) and bool(wide0[:, H + 1:].isnan().all())
    assert bool((both[..., :off] == 7).all()) and bool((both[..., off + H:] == 7).all())
    p = view.detach().requires_grad_()
    hh, ll = gated_scan(p, start.cuda())
    g = torch.autograd.grad((hh, ll), p, (dh[:1, :1].cuda().expand(B, T, H), torch.ones((), device="cuda").expand(B, H)))[0]
    ref = SO.gated_scan(_np(pre), _np(start), None, False, np.broadcast_to(_np(dh[:1, :1]), (B, T, H)), np.ones((B, H)), need_grad=True)
    _check(g, ref["dpre"], ref["dpre_err"], "dpre")
    g = torch.autograd.grad(gated_scan(p)[0].float().sum(), p)[0]       # a gradient from the states alone
    ref = SO.gated_scan(_np(pre), None, None, False, np.ones((B, T, H)), None, need_grad=True)
    _check(g, ref["dpre"], ref["dpre_err"], "dpre")


@pytest.mark.parametrize("B,T,H", [(1, 30000, 96), (40, 2000, 64), (3, 5000, 300)])
def test_gated_scan_gives_the_same_bits_every_time(B, T, H):
    """fp32 results do not depend on which blocks of a sequence finish first: calls alone, back to back and next to another stream's."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, dlast = _scan_inputs(B, T, H, F32, False, "rows", seed=B, gate=(-5.0, 1.0))
    p, s, dl = pre.cuda().requires_grad_(), start.cuda().requires_grad_(), dlast.cuda()

    def one():
        h, last = gated_scan(p, s)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (p, s), (torch.ones_like(h), dl))
    want = one()
    torch.cuda.synchronize()
    side, noise = torch.cuda.Stream(), torch.empty(1 << 26, device="cuda")
    for r in range(12):
        if r > 5:
            with torch.cuda.stream(side):
                noise.mul_(1.5)
        assert all(torch.equal(a, b) for a, b in zip(one(), want)), r


def test_gated_scan_gradient_from_final_state_alone():
    from spot_amd.recurrence import gated_scan
    for T in (1, 5, 200):
        pre, start, lengths, _, dlast = _scan_inputs(3, T, 20, F32, True, "rows", seed=T)
        p, s = pre.cuda().requires_grad_(), start.cuda().requires_grad_()
        g = torch.autograd.grad(gated_scan(p, s, lengths.cuda())[1], (p, s), dlast.cuda())
        ref = SO.gated_scan(_np(pre), _np(start), _np(lengths), False, None, _np(dlast), need_grad=True)
        _check(g[0], ref["dpre"], ref["dpre_err"], "dpre")
        _check(g[1], ref["dh0"], ref["dh0_err"], "dh0")


@pytest.mark.parametrize("T", [30, 700])
def test_gated_scan_backward_twice_and_captured_apart_from_its_forward(T):
    """The second backward pass through a graph, and a captured one that is replayed without its forward, give the bits of the first."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, dh, dlast = _scan_inputs(2, T, 96, BF, False, "rows", seed=T)
    d, dl = dh.cuda(), dlast.cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        p, s = pre.cuda().requires_grad_(), start.cuda().requires_grad_()
        y = gated_scan(p, s)
        first = torch.autograd.grad(y, (p, s), (d, dl), retain_graph=True)
        again = torch.autograd.grad(y, (p, s), (d, dl), retain_graph=True)
        z = gated_scan(p, s)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            out = torch.autograd.grad(z, (p, s), (d, dl), retain_graph=True)
        for _ in range(3):
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(first, out))
            out[0].zero_()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gated_scan_gradient_against_differences():
    from spot_amd.recurrence import gated_scan
    pre, start, lengths, dh, dlast = _scan_inputs(3, 150, 24, F32, True, "shared", seed=3)
    p, s = pre.cuda().requires_grad_(), start.cuda().requires_grad_()
    value = lambda a, b: (lambda r: (r[0].double() * dh.cuda()).sum() + (r[1].double() * dlast.cuda()).sum())(gated_scan(a, b, lengths.cuda()))  # noqa: E731
    gp, gs = torch.autograd.grad(value(p, s), (p, s))
    g = torch.Generator().manual_seed(9)
    vp, vs = torch.randn(pre.shape, generator=g).cuda(), torch.randn(24, generator=g).cuda()
    e = 2.0 ** -7
    with torch.no_grad():
        slope = float((value(p + e * vp, s + e * vs) - value(p - e * vp, s - e * vs)) / (2 * e))
        far = float((value(p + 2 * e * vp, s + 2 * e * vs) - value(p - 2 * e * vp, s - 2 * e * vs)) / (4 * e))
    got = float((gp.double() * vp).sum() + (gs.double() * vs).sum())
    # the truncation error of the step e is a third of the change from step 2e to e; fp32 rounding of 10,800 states of order 1 with
    # random signs under gradients of order 1 is 104 * 1e-6 in the value, 1e-4 / e in the slope
    assert abs(got - slope) <= abs(slope - far) + 2e-2, (got, slope, far)


def test_gated_scan_frames_one_by_one_continue_the_sequence():
    """Whole sequence = parts of any length with the state handed on = one frame at a time with the state in place."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(5, 300, 48, BF, False, "rows", seed=2)
    p = pre.cuda()
    ref = SO.gated_scan(_np(pre), _np(start))
    state, parts = start.cuda(), []
    for lo, hi in ((0, 1), (1, 1), (1, 130), (130, 300)):
        h, state = gated_scan(p[:, lo:hi], state)
        parts.append(h)
    _check(torch.cat(parts, 1), ref["h"], ref["h_err"], "h in parts")
    _check(state, ref["last"], ref["last_err"], "last in parts")
    state, out = start.cuda(), torch.empty(5, 300, 48, dtype=BF, device="cuda")
    for t in range(300):
        _, s = gated_scan(p[:, t:t + 1], state, out=out[:, t:t + 1], state_out=state)
        assert s.data_ptr() == state.data_ptr()
    _check(out, ref["h"], ref["h_err"], "h frame by frame")
    _check(state, ref["last"], ref["last_err"], "last frame by frame")


def test_gated_scan_equals_the_short_clip_kernels():
    """On clips the operator and stes_mingru_scan_fwd / _bwd are the same recurrence (the latter reads the stored bf16 states)."""
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    B, T, H = 4, 64, 768
    pre, start, _, dh, _ = _scan_inputs(B, T, H, BF, False, "shared", seed=11)
    p, s = pre.cuda(), start.cuda()
    h, dpre = torch.empty(B, T, H, dtype=BF, device="cuda"), torch.empty(B, T, 2 * H, dtype=BF, device="cuda")
    d32 = dh.float().cuda()
    lib.call("stes_mingru_scan_fwd", lib.ptr(p), lib.ptr(s), lib.ptr(h), B, T, H)
    lib.call("stes_mingru_scan_bwd", lib.ptr(p), lib.ptr(s), lib.ptr(h), lib.ptr(d32), H, lib.ptr(dpre), B, T, H)
    q = p.clone().requires_grad_()
    h2, _ = gated_scan(q, s)
    g = torch.autograd.grad(h2, q, dh.cuda())[0]
    err = SO.gated_scan(_np(pre), _np(start))["h_err"]
    _check(h2, _np(h), 2 * err + 2.0 ** -8 * np.abs(_np(h)), "h")
    # its states carry 2^-8 of their size from storage, which enters d gate times |l| z a <= |d cand| / 4 + ... : a loose common bound
    assert float((g.float() - dpre.float()).abs().max()) <= 2.0 ** -6 * float(dpre.float().abs().max())


@pytest.mark.parametrize("shape", [(0, 5, 8), (3, 0, 8), (3, 5, 0), (0, 0, 0)])
def test_gated_scan_empty(shape):
    from spot_amd.recurrence import gated_scan
    B, T, W = shape
    H = W // 2
    for h0 in (None, torch.randn(B, H).cuda(), torch.randn(H).cuda()):
        pre = torch.randn(B, T, W).cuda().requires_grad_()
        s = None if h0 is None else h0.requires_grad_()
        h, last = gated_scan(pre, s)
        assert h.shape == (B, T, H) and last.shape == (B, H)
        if T == 0 or H == 0:
            assert torch.equal(last, torch.zeros(B, H, device="cuda") if s is None else s.expand(B, H))
        g = torch.autograd.grad((h, last), (pre,) if s is None else (pre, s), (torch.ones_like(h), torch.full_like(last, 2.0)))
        assert g[0].shape == pre.shape
        if s is not None:
            assert g[1].shape == s.shape and (T or B or H) is not None
            if T == 0:
                assert torch.equal(g[1], torch.full_like(s, 2.0 if s.dim() == 2 else 2.0 * B))


def test_gated_scan_offsets_beyond_32_bits():
    """Sequences more than 2^31 elements apart, and frames more than 2^31 elements into a sequence."""
    from spot_amd.recurrence import gated_scan
    T, H = 200, 64
    base = torch.zeros((1 << 31) + (1 << 20), dtype=BF, device="cuda")
    pre, start, _, dh, _ = _scan_inputs(2, T, H, BF, False, "rows", seed=4)
    far = base.as_strided((2, T, 2 * H), ((1 << 31) + 64, 2 * H, 1))
    far.copy_(pre.cuda())
    want, wl = gated_scan(pre.cuda(), start.cuda())
    h, last = gated_scan(far, start.cuda())
    assert torch.equal(h, want) and torch.equal(last, wl)
    step = (1 << 31) // (T - 1) // 64 * 64 + 64                          # frame T-1 starts beyond element 2^31
    far = base.as_strided((1, T, 2 * H), (0, step, 1))
    far.copy_(pre[:1].cuda())
    p = far.detach().requires_grad_()
    h, last = gated_scan(p, start[:1].cuda())
    assert torch.equal(h, want[:1]) and torch.equal(last, wl[:1])
    q = pre[:1].cuda().requires_grad_()
    ga, = torch.autograd.grad(gated_scan(q, start[:1].cuda())[0], q, dh[:1].cuda())
    gb, = torch.autograd.grad(h, p, dh[:1].cuda())
    assert torch.equal(ga, gb)


def test_gated_scan_long_sequence_equals_its_parts():
    """300,000 frames (460 MB): the last frames against a call that starts from the state in front of them."""
    from spot_amd.recurrence import gated_scan
    g = torch.Generator(device="cuda").manual_seed(0)
    pre = torch.randn(1, 300000, 2 * 768, device="cuda", generator=g, dtype=BF)
    pre[..., :768] -= 4
    h, last = gated_scan(pre)
    _, s = gated_scan(pre[:, :299000])
    h2, last2 = gated_scan(pre[:, 299000:], s)
    # two associations of the same sums: twice the oracle's bound at a memory of some 60 frames (60 * 20 u * |c| <= 5), and one step of bf16
    assert float((last - last2).abs().max()) <= 2 * 60 * 20 * SO.U * 5
    assert float((h[:, 299000:].float() - h2.float()).abs().max()) <= 2 * 60 * 20 * SO.U * 5 + 2.0 ** -7 * float(h2.float().abs().max())


@pytest.mark.parametrize("T", [1, 64, 1000])
def test_gated_scan_on_another_stream_and_two_calls_at_once(T):
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(4, T, 768, BF, False, "rows", seed=T)
    p, s = pre.cuda(), start.cuda()
    want, wl = gated_scan(p, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(gated_scan(p, s))
    torch.cuda.synchronize()
    for h, last in got:
        assert torch.equal(h, want) and torch.equal(last, wl)


def test_gated_scan_calls_of_changing_sizes_share_a_stream():
    """Calls of growing and shrinking sizes one after the other on one stream (they take two kept workspaces in turn), forward and
    backward, from two threads at once, next to a captured call that is replayed among them."""
    import threading
    from spot_amd.recurrence import gated_scan
    sizes = [(1, 300, 64), (3, 1000, 200), (1, 257, 8), (2, 5000, 64), (1, 300, 64), (4, 600, 130), (1, 20000, 8), (3, 1000, 200)]
    inputs = [_scan_inputs(B, T, H, BF, False, "rows", seed=T + H)[:2] for B, T, H in sizes]
    inputs = [(a.cuda().requires_grad_(), b.cuda()) for a, b in inputs]

    def one(i):
        p, s = inputs[i]
        h, last = gated_scan(p, s)
        return h.detach(), last.detach(), torch.autograd.grad(h, p, torch.ones_like(h))[0]
    want = []
    for i in range(len(sizes)):
        p, s = inputs[i]
        with torch.cuda.stream(torch.cuda.Stream()):                    # a stream of its own: workspaces of its own
            want.append(one(i))
        torch.cuda.synchronize()
    cap = inputs[1][0].detach()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = gated_scan(cap, inputs[1][1])
    bad = []

    def work(seed):
        with torch.cuda.stream(shared):
            for i in np.random.default_rng(seed).integers(0, len(sizes), 40):
                bad.extend([i] if not all(torch.equal(a, b) for a, b in zip(one(i), want[i])) else [])
    shared = torch.cuda.Stream()
    shared.wait_stream(torch.cuda.current_stream())
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for _ in range(5):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[1][0]) and torch.equal(out[1], want[1][1])
    for t in threads:
        t.join(100)
    assert not bad


def test_gated_scan_keeps_workspaces_of_few_streams():
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    pre, start, _, _, _ = _scan_inputs(2, 900, 96, BF, False, "rows", seed=8)
    p, s = pre.cuda(), start.cuda()
    want = gated_scan(p, s)
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in range(6)]
    most = lib.native().keep_streams(3)
    try:
        for _ in range(12):
            for st in streams:
                with torch.cuda.stream(st):
                    got.append(gated_scan(p, s))
            assert lib.native().kept_streams() <= max(3, most)
    finally:
        lib.native().keep_streams(most)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.parametrize("T", [1, 64, 700])
def test_gated_scan_in_graphs(T):
    """Forward and backward captured, replayed several times with new inputs and eager work in between, next to a second graph of the
    same memory pool."""
    from spot_amd.recurrence import gated_scan
    pre, start, _, dh, dlast = _scan_inputs(2, T, 96, BF, False, "rows", seed=T + 1)
    p, s = pre.cuda().requires_grad_(), start.cuda().requires_grad_()
    d, dl = dh.cuda(), dlast.cuda()

    def work():
        h, last = gated_scan(p, s)
        return (h, last) + torch.autograd.grad((h, last), (p, s), (d, dl))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, gr in enumerate(graphs):
        with torch.cuda.graph(gr, pool=None if i == 0 else graphs[0].pool()):
            outs.append(work())
    for r in range(4):
        with torch.no_grad():
            p.copy_(torch.roll(p, 1, 1) * (1.0 if r else 0.5))
            s.mul_(0.5)
        want = [t.detach().clone() for t in work()]
        for gr, out in zip(graphs, outs):
            for t in out:
                t.detach().fill_(NAN)
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def _differentiable_calls():
    """(leaf, call of it) for both operators, with kept statistics and, for the scan, joined blocks."""
    from spot_amd.distill import topk_distill_loss
    from spot_amd.recurrence import gated_scan
    p = torch.randn(2, 300, 16, device="cuda", requires_grad=True)
    x = torch.randn(9, 50, device="cuda", requires_grad=True)
    val, idx = torch.randn(9, 50, device="cuda").topk(3)
    n = torch.tensor([300, 17], dtype=torch.int32, device="cuda")
    return [(p, lambda t: gated_scan(t, lengths=n)[0].square().sum()), (x, lambda t: topk_distill_loss(t, idx, val, 2.0))]


def test_gradients_behave_as_torchs_own_functions_do():
    """Kept graphs, graphs used up, inputs changed in between, tensors saved elsewhere, recomputation, gradients that accumulate, hooks,
    anomaly mode, no second derivative and no tangents, and no memory that stays."""
    from spot_amd import lib
    for leaf, f in _differentiable_calls():
        want, = torch.autograd.grad(f(leaf), leaf)
        y = f(leaf)
        a, = torch.autograd.grad(y, leaf, retain_graph=True)
        b, = torch.autograd.grad(y, leaf)
        assert torch.equal(a, want) and torch.equal(b, want)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf)
        c = leaf.detach().clone().requires_grad_()
        d = c * 1.0
        y = f(d)
        d.data.add_(0)                                      # (not seen by autograd, and it changes nothing)
        torch.autograd.grad(y, c, retain_graph=True)
        with torch.no_grad():
            d.add_(1.0)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, c)
        with torch.autograd.graph.save_on_cpu():
            y = f(leaf)
        assert torch.equal(torch.autograd.grad(y, leaf)[0], want)
        again = torch.utils.checkpoint.checkpoint(f, leaf, use_reentrant=False)
        assert torch.equal(torch.autograd.grad(again, leaf)[0], want)
        seen = []
        with torch.autograd.set_detect_anomaly(True):
            y = f(leaf)
            y.register_hook(lambda g: seen.append(g) or 2 * g)
            y.backward()
            f(leaf).backward()
        assert len(seen) == 1
        _check(leaf.grad, 3 * _np(want), 8 * SO.U * np.abs(_np(want)), "accumulated")
        g, = torch.autograd.grad(f(leaf), leaf, create_graph=True)
        _check(g, _np(want), 0 * np.abs(_np(want)), "create_graph")
        with pytest.raises(RuntimeError):
            torch.autograd.grad((g * leaf).sum(), leaf)
        y = f(leaf)
        up = torch.ones_like(y, requires_grad=True)
        g, = torch.autograd.grad(y, leaf, up, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad((g * leaf * up).sum(), up)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(lib.StesError):
                f(torch.autograd.forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf)))
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(leaf.detach())
        with pytest.raises(RuntimeError):
            torch.vmap(f)(torch.stack([leaf.detach()] * 2))
        leaf.grad = None
        torch.cuda.synchronize()
        del y, again, g, a, b, c, d, seen
        f(leaf)
        before = torch.cuda.memory_allocated()
        for i in range(50):
            y = f(leaf)
            if i % 2:
                torch.autograd.grad(y, leaf)
            del y
        assert torch.cuda.memory_allocated() == before


def test_backward_passes_from_several_threads():
    import threading
    for leaf, f in _differentiable_calls():
        want, = torch.autograd.grad(f(leaf), leaf)
        torch.cuda.synchronize()
        got = []

        def work():
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got.append(torch.autograd.grad(f(leaf), leaf)[0])
                torch.cuda.current_stream().synchronize()
        threads = [threading.Thread(target=work) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        torch.cuda.synchronize()
        assert len(got) == 80 and all(torch.equal(g, want) for g in got)


def test_capture_refuses_leaves_that_an_eager_graph_holds():
    """A backward pass captured while an eager autograd graph of the same leaf lives would end the process: the captured forward refuses."""
    from spot_amd import lib
    from spot_amd.distill import topk_distill_loss
    from spot_amd.recurrence import gated_scan
    p = torch.randn(2, 4, 16, device="cuda", requires_grad=True)
    i, v = torch.zeros(8, 1, dtype=torch.int64, device="cuda"), torch.zeros(8, 1, device="cuda")
    x = torch.randn(8, 5, device="cuda", requires_grad=True)
    for leaf, call in ((p, lambda: gated_scan(p)[0]), (x, lambda: topk_distill_loss(x, i, v))):
        alive = call()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with pytest.raises(lib.StesError):
            with torch.cuda.graph(gr):
                torch.ones(4, device="cuda").mul_(2)
                call()
        del alive
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = call()
            g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        gr.replay()
        torch.cuda.synchronize()
        z = call()
        assert torch.equal(y, z) and torch.equal(g, torch.autograd.grad(z, leaf, torch.ones_like(z))[0])


def test_gated_scan_refusals():
    from spot_amd import lib
    from spot_amd.recurrence import gated_scan
    p = torch.zeros(2, 3, 8, device="cuda")
    bad = [dict(pre=torch.zeros(2, 3, 7, device="cuda")), dict(pre=p.half()), dict(pre=p[0]), dict(pre=p.transpose(1, 2)),
           dict(pre=p[:, :1].expand(2, 3, 8)), dict(h0=torch.zeros(2, 4)), dict(h0=torch.zeros(2, 4, device="cuda", dtype=BF)),
           dict(h0=torch.zeros(3, 4, device="cuda")), dict(lengths=torch.zeros(2, dtype=torch.int64, device="cuda")),
           dict(lengths=torch.zeros(2, dtype=torch.int32)), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
           dict(out=torch.zeros(2, 3, 4, device="cuda", dtype=BF)), dict(out=torch.zeros(2, 3, 5, device="cuda")),
           dict(out=torch.zeros(2, 1, 4, device="cuda").expand(2, 3, 4)),
           dict(out=torch.zeros(1, 3, 4, device="cuda").expand(2, 3, 4)),
           dict(state_out=torch.zeros(4, device="cuda")), dict(state_out=torch.zeros(1, 4, device="cuda").expand(2, 4)),
           dict(pre=p.clone().requires_grad_(), out=torch.zeros(2, 3, 4, device="cuda"))]
    shared = torch.zeros(8, device="cuda")
    bad.append(dict(h0=shared[:4], state_out=shared.view(2, 4)))
    for kw in bad:
        with pytest.raises(lib.StesError):
            gated_scan(**{"pre": p, **kw})
    q = p.clone().requires_grad_()
    h, _ = gated_scan(q)
    g, = torch.autograd.grad(h.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ----------------------------------------------------------------------------------------------------- distillation
def _kl_inputs(M, V, k, dtype, seed, holes=False, weighted=False):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(M, V, generator=g) * 3
    s = (0.7 * t + 1.5 * torch.randn(M, V, generator=g)).to(dtype)
    val, idx = t.topk(min(k, V), 1)
    if holes:
        idx[torch.rand(idx.shape, generator=g) < 0.2] = -1
        idx[::5] = -1
    w = torch.rand(M, generator=g) + 0.5 if weighted else None
    if weighted:
        w[1::7] = 0.0
    return s, idx, val, w


def _kl_compare(s, idx, val, w, tau, denom=None, up=1.0):
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    d = lambda t: None if t is None else t.cuda()  # noqa: E731
    ref = SO.topk_distill(_np(s), _np(idx), _np(val), tau, _np(w), denom, scale=up)
    x = s.cuda().requires_grad_()
    loss = topk_distill_loss(x, d(idx), d(val), tau, d(w), denom)
    g, = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    _check(loss, ref["loss"], ref["loss_err"], "loss")
    _check(g, ref["dlogits"], ref["dlogits_err"], "dlogits")
    l2, g2 = topk_distill_grad(s.cuda(), d(idx), d(val), tau, d(w), denom, grad_scale=up)
    _check(l2, ref["loss"], ref["loss_err"], "loss in one pass")
    _check(g2, ref["dlogits"], ref["dlogits_err"], "dlogits in one pass")
    with torch.no_grad():
        assert torch.equal(topk_distill_loss(x, d(idx), d(val), tau, d(w), denom), l2) and torch.equal(l2, loss)
    l3, g3 = topk_distill_grad(s.cuda(), d(idx), d(val), tau, d(w), denom, grad_scale=up)
    assert torch.equal(l2, l3) and torch.equal(g2, g3)
    return ref


KL_CASES = [  # M, V, k, dtype, tau, holes, weighted
    (1, 1, 1, F32, 1.0, False, False), (1, 2, 1, BF, 2.0, False, True), (5, 2, 2, F32, 0.5, True, False), (33, 7, 4, F32, 1.0, True, True),
    (1024, 7, 4, F32, 1.0, True, True), (9, 8, 8, BF, 1.0, False, False), (17, 33, 5, BF, 4.0, True, False), (6, 64, 64, F32, 1.0, False, True),
    (5, 65, 40, BF, 2.0, True, True), (70, 129, 16, F32, 1.5, False, False), (7, 255, 3, BF, 1.0, True, True), (13, 256, 20, F32, 1.0, True, False),
    (4, 511, 33, BF, 2.0, False, True), (4, 513, 2, F32, 2.0, True, False), (9, 1000, 16, BF, 2.0, True, True), (3, 2049, 64, F32, 1.0, False, False),
    (5, 4095, 10, BF, 1.0, True, False), (3, 4097, 10, BF, 1.0, True, True), (3, 8191, 64, F32, 3.0, True, True), (2, 16385, 7, BF, 1.0, False, False),
    (2, 32003, 32, BF, 2.0, True, True), (2, 50001, 64, F32, 1.0, False, True), (2, 65537, 5, BF, 1.0, True, False), (1, 140001, 8, F32, 1.0, False, False),
    (1, 300007, 64, BF, 2.0, False, False),
]


@pytest.mark.parametrize("M,V,k,dtype,tau,holes,weighted", KL_CASES)
def test_distill_loss_and_gradient(M, V, k, dtype, tau, holes, weighted):
    _kl_compare(*_kl_inputs(M, V, k, dtype, M + V, holes, weighted), tau, denom=None if M % 2 else 3.5, up=0.75)


@pytest.mark.parametrize("V", [7, 300, 5000, 70001])
def test_distill_index_and_value_types_duplicates_and_order(V):
    s, idx, val, w = _kl_inputs(6, V, 5, F32, V, False, True)
    idx[0, 3] = idx[0, 1]                                                # a class listed twice, and three times
    idx[1, :3] = idx[1, 4]
    idx[2] = idx[2].flip(0)
    val[3, 2:] = -INF                                                    # listed, with no probability
    idx[4, 0], idx[4, 1] = 0, V - 1                                      # the ends of a row
    _kl_compare(s, idx, val, w, 2.0)
    _kl_compare(s, idx.int(), val, w, 2.0)
    _kl_compare(s, idx.int(), val.to(BF), w, 2.0)
    wide_i, wide_v = torch.full((6, 9), -7).long(), torch.full((6, 9), NAN)
    wide_i[:, 2:7], wide_v[:, 2:7] = idx, val
    from spot_amd.distill import topk_distill_grad
    a = topk_distill_grad(s.cuda(), wide_i.cuda()[:, 2:7], wide_v.cuda()[:, 2:7], 2.0, w.cuda())
    b = topk_distill_grad(s.cuda(), idx.cuda(), val.cuda(), 2.0, w.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("V", [6, 700, 9000, 80000])
def test_distill_rows_that_do_not_count(V):
    """Rows of weight zero, rows that list nothing and rows whose every listed value is -inf: zero loss and zero gradient, whatever
    their logits hold (NaN, infinities, the type's lowest value)."""
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, idx, val, _ = _kl_inputs(7, V, 3, F32, V)
    w = torch.ones(7)
    idx[0], val[1], w[2] = -1, -INF, 0.0
    idx[6, 1:] = -1
    val[6, 1:] = NAN                                                     # values of unused places are not looked at
    dirty = s.clone()
    dirty[0], dirty[1], dirty[2] = NAN, INF, torch.finfo(F32).min
    ref = SO.topk_distill(_np(s), _np(idx), np.nan_to_num(_np(val), nan=0.0, neginf=-np.inf), 1.0, _np(w))
    x = dirty.cuda().requires_grad_()
    loss = topk_distill_loss(x, idx.cuda(), val.cuda(), weight=w.cuda())
    _check(loss, ref["loss"], ref["loss_err"], "loss")
    g, = torch.autograd.grad(loss, x)
    l2, g2 = topk_distill_grad(dirty.cuda(), idx.cuda(), val.cuda(), weight=w.cuda())
    for t in (g, g2):
        _check(t, ref["dlogits"], ref["dlogits_err"], "dlogits")
        assert not bool(t[:3].any())
    none = topk_distill_grad(dirty.cuda(), torch.full_like(idx, -1).cuda(), val.cuda())
    assert float(none[0]) == 0.0 and not bool(none[1].any())


@pytest.mark.parametrize("V", [6, 700, 9000, 80000])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_distill_masked_classes_and_extreme_logits(V, dtype):
    """Classes masked with -inf or with the type's lowest value have q = 0; a listed class of q = 0 makes the loss infinite; rows at the lowest
    value throughout are uniform; NaN, +inf and a whole row of -inf give NaN rows."""
    from spot_amd.distill import topk_distill_grad
    s, idx, val, _ = _kl_inputs(6, V, 2, dtype, V + 1)
    low = torch.finfo(dtype).min
    for row, m in ((0, -INF), (1, low)):
        keep = torch.zeros(V, dtype=torch.bool)
        keep[idx[row]] = True
        s[row, ~keep] = m
    s[2] = low
    finite = torch.tensor([0, 1, 2, 5])
    _kl_compare(s[finite], idx[finite], val[finite], None, 0.5)
    s[3, idx[3, 0]] = -INF                                               # the teacher's best class is impossible for the student
    loss, g = topk_distill_grad(s.cuda(), idx.cuda(), val.cuda())
    assert float(loss) == INF and bool(g.isfinite().all())
    for v in (NAN, INF):
        t = s.clone()
        t[4, V // 2] = v
        loss, g = topk_distill_grad(t.cuda(), idx.cuda(), val.cuda())
        assert bool(loss.isnan()) and bool(g[4].isnan().all()) and bool(g[:4].isfinite().all()) and bool(g[5].isfinite().all())
    t = s.clone()
    t[4] = -INF
    loss, g = topk_distill_grad(t.cuda(), idx.cuda(), val.cuda())
    assert bool(loss.isnan()) and bool(g[4].isnan().all()) and bool(g[5].isfinite().all())


@pytest.mark.parametrize("V", [6, 700, 9000, 80000])
def test_distill_index_beyond_the_classes_gives_nan_and_touches_nothing_else(V):
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, idx, val, _ = _kl_inputs(4, V, 3, F32, V)
    for bad in (V, V + 1, (1 << 31) - 1, 1 << 40):
        i = idx.clone()
        i[2, 1] = bad
        x = s.cuda().requires_grad_()
        loss = topk_distill_loss(x, i.cuda(), val.cuda())
        g, = torch.autograd.grad(loss, x)
        l2, g2 = topk_distill_grad(s.cuda(), i.cuda(), val.cuda())
        for a, b in ((loss, g), (l2, g2)):
            assert bool(a.isnan()) and bool(b[2].isnan().all()) and bool(b[[0, 1, 3]].isfinite().all())


@pytest.mark.parametrize("V,pad", [(7, 1), (7, 0), (700, 3), (9000, 8), (9001, 5), (70000, 1)])
@pytest.mark.parametrize("sdt,ddt", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
def test_distill_output_types_strides_and_accumulation(V, pad, sdt, ddt):
    from spot_amd.distill import topk_distill_grad
    M = 5
    s, idx, val, w = _kl_inputs(M, V, 4, sdt, V, True, True)
    ref = SO.topk_distill(_np(s), _np(idx), _np(val), 1.0, _np(w))
    wide = torch.full((M, V + 2 * pad), NAN, dtype=sdt).cuda()
    wide[:, pad:pad + V] = s.cuda()
    out = torch.full((M, V + pad), 7.0, dtype=ddt).cuda()
    loss, g = topk_distill_grad(wide[:, pad:pad + V], idx.cuda(), val.cuda(), weight=w.cuda(), out=out[:, :V])
    _check(loss, ref["loss"], ref["loss_err"], "loss")
    _check(g, ref["dlogits"], ref["dlogits_err"], "dlogits")
    assert bool((out[:, V:] == 7).all()) and bool(wide[:, :pad].isnan().all())
    old = (torch.randn(M, V + pad, generator=torch.Generator().manual_seed(1)) * 1e-2).to(ddt)
    out = old.cuda()
    topk_distill_grad(wide[:, pad:pad + V], idx.cuda(), val.cuda(), weight=w.cuda(), out=out[:, :V], accumulate=True)
    o = _np(old)
    total = o[:, :V] + ref["dlogits"]
    _check(out[:, :V], total, ref["dlogits_err"] + 2 * SO.U * (np.abs(total) + np.abs(o[:, :V])), "accumulated")
    assert torch.equal(out[:, V:].cpu(), old[:, V:])
    dead = (idx < 0).all(1) | (w == 0)
    assert torch.equal(out.cpu()[dead], old[dead])


def test_distill_leading_dimensions_and_empty():
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, idx, val, w = _kl_inputs(12, 7, 4, F32, 1, True, True)
    a = topk_distill_grad(s.view(3, 4, 7).cuda(), idx.view(3, 4, 4).cuda(), val.view(3, 4, 4).cuda(), weight=w.view(3, 4).cuda())
    b = topk_distill_grad(s.cuda(), idx.cuda(), val.cuda(), weight=w.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1].view(12, 7), b[1])
    x = s.view(3, 4, 7).cuda().requires_grad_()
    g, = torch.autograd.grad(topk_distill_loss(x, idx.view(3, 4, 4).cuda(), val.view(3, 4, 4).cuda(), weight=w.view(3, 4).cuda()), x)
    _check(g.view(12, 7), _np(b[1]), 4 * SO.U * np.abs(_np(b[1])), "leading dimensions")
    e = torch.zeros(0, 7, device="cuda", requires_grad=True)
    loss = topk_distill_loss(e, torch.zeros(0, 2, dtype=torch.int64, device="cuda"), torch.zeros(0, 2, device="cuda"))
    assert float(loss) == 0.0 and torch.autograd.grad(loss, e)[0].shape == (0, 7)
    assert float(topk_distill_grad(e, torch.zeros(0, 2, dtype=torch.int64, device="cuda"), torch.zeros(0, 2, device="cuda"))[0]) == 0.0


@pytest.mark.parametrize("V", [6, 300, 5000, 40000, 200000])
def test_distill_one_row_and_views(V):
    """A single row without a leading dimension, transposed and expanded logits: copies where the kernels need them."""
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, idx, val, w = _kl_inputs(4, V, 3, F32, V + 7, False, True)
    ref = SO.topk_distill(_np(s[:1]), _np(idx[:1]), _np(val[:1]), 2.0, _np(w[:1]))
    loss, g = topk_distill_grad(s[0].cuda(), idx[0].cuda(), val[0].cuda(), 2.0, w[0].cuda())
    _check(loss, ref["loss"], ref["loss_err"], "one row")
    _check(g[None], ref["dlogits"], ref["dlogits_err"], "one row")
    want = topk_distill_grad(s.cuda(), idx.cuda(), val.cuda(), 2.0, w.cuda())
    x = s.t().contiguous().cuda().requires_grad_()
    loss = topk_distill_loss(x.t(), idx.t().contiguous().cuda().t(), val.t().contiguous().cuda().t(), 2.0, w.cuda())
    g, = torch.autograd.grad(loss, x)
    assert torch.equal(loss, want[0])
    _check(g.t(), _np(want[1]), 4 * SO.U * np.abs(_np(want[1])), "transposed")
    y = s[:1].cuda().requires_grad_()
    loss = topk_distill_loss(y.expand(4, V), idx[:1].cuda().expand(4, 3), val[:1].cuda().expand(4, 3), 2.0, w.cuda())
    g, = torch.autograd.grad(loss, y)
    ref = SO.topk_distill(_np(s[:1]).repeat(4, 0), _np(idx[:1]).repeat(4, 0), _np(val[:1]).repeat(4, 0), 2.0, _np(w))
    _check(loss, ref["loss"], ref["loss_err"], "expanded")
    total = ref["dlogits"].sum(0, keepdims=True)
    _check(g, total, ref["dlogits_err"].sum(0, keepdims=True) + 4 * SO.U * np.abs(ref["dlogits"]).sum(0, keepdims=True), "expanded")


def test_distill_calls_of_changing_sizes_share_a_stream():
    """Calls with few and many workgroups one after the other, on two streams at once: each finds the words clean through which
    workgroups hand over their sums."""
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    cases = []
    for M, V, k in ((1024, 7, 4), (1, 7, 4), (3, 20000, 5), (5000, 600, 3), (20000, 530, 2), (70, 300, 64), (1024, 7, 4), (300, 4000, 16), (2000, 2, 1)):
        s, idx, val, _ = _kl_inputs(M, V, k, BF, M + V)
        ref = SO.topk_distill(_np(s), _np(idx), _np(val), 2.0)
        cases.append((s.cuda(), idx.cuda(), val.cuda(), ref))
    got, order = [], np.random.default_rng(0).integers(0, len(cases), 60)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in order:
        s, idx, val, _ = cases[i]
        for st in streams:
            with torch.cuda.stream(st):
                got.append((i, topk_distill_loss(s, idx, val, 2.0), topk_distill_grad(s, idx, val, 2.0)[0]))
    torch.cuda.synchronize()
    for i, a, b in got:
        _check(a, cases[i][3]["loss"], cases[i][3]["loss_err"], "loss")
        assert torch.equal(a, b)


def test_distill_gradient_against_differences():
    from spot_amd.distill import topk_distill_loss
    s, idx, val, w = _kl_inputs(64, 40, 6, F32, 3, True, True)
    x, i, v, ww = s.cuda().requires_grad_(), idx.cuda(), val.cuda(), w.cuda()
    f = lambda t: topk_distill_loss(t, i, v, 2.0, ww)  # noqa: E731
    g, = torch.autograd.grad(f(x), x)
    d = torch.randn(64, 40, generator=torch.Generator().manual_seed(2)).cuda()
    e = 2.0 ** -5
    with torch.no_grad():
        slope, far = (float((f(x + r * d) - f(x - r * d)).double() / (2 * r)) for r in (e, 2 * e))
    # truncation: a third of the change from 2e to e; the loss, of order 4, is rounded to fp32: 2 * 2.4e-7 * 4 / (2 e) = 3e-5
    assert abs(float((g.double() * d).sum()) - slope) <= abs(slope - far) + 6e-5


def test_distill_rows_beyond_32_bits():
    from spot_amd.distill import topk_distill_grad
    s, idx, val, _ = _kl_inputs(3, 1000, 8, BF, 0)
    base = torch.zeros((1 << 31) + 4096, dtype=BF, device="cuda")
    far = base.as_strided((3, 1000), (1 << 30, 1))
    far.copy_(s.cuda())
    out = torch.zeros((1 << 31) + 4096, dtype=BF, device="cuda").as_strided((3, 1000), (1 << 30, 1))
    a = topk_distill_grad(far, idx.cuda(), val.cuda(), out=out)
    b = topk_distill_grad(s.cuda(), idx.cuda(), val.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("M,V", [(50, 7), (600, 40), (40, 3000)])
def test_distill_streams_and_graphs(M, V):
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, idx, val, w = _kl_inputs(M, V, 4, F32, 5, True, True)
    x, i, v, ww = s.cuda().requires_grad_(), idx.cuda(), val.cuda(), w.cuda()

    def work():
        loss = topk_distill_loss(x, i, v, 2.0, ww)
        return (loss, torch.autograd.grad(loss, x)[0]) + topk_distill_grad(x, i, v, 2.0, ww)
    want = [t.detach().clone() for t in work()]
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(st):
            got.append(work())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    del got, r
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for n, gr in enumerate(graphs):
        with torch.cuda.graph(gr, pool=None if n == 0 else graphs[0].pool()):
            outs.append(work())
    for r in range(4):
        with torch.no_grad():
            x.copy_(torch.roll(x, 1, 0) * (0.5 if r == 0 else 1.0))
        want = [t.detach().clone() for t in work()]
        for gr, out in zip(graphs, outs):
            for t in out:
                t.detach().fill_(NAN)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_distill_refusals():
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    s, i, v = torch.zeros(4, 7, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, 2, device="cuda")
    for kw in (dict(logits=s.half()), dict(idx=i.short()), dict(idx=i[:3]), dict(idx=i.cpu()), dict(val=v.double()), dict(val=v[:, :1]),
               dict(idx=i.repeat(1, 40), val=v.repeat(1, 40)), dict(idx=i[:, :0], val=v[:, :0]), dict(temperature=0.0), dict(temperature=-1),
               dict(temperature=NAN), dict(temperature=INF), dict(temperature=1e-40), dict(denom=0.0), dict(denom=-2.0), dict(denom=NAN), dict(weight=torch.ones(4)),
               dict(weight=torch.ones(3, device="cuda")), dict(weight=torch.ones(4, device="cuda", dtype=BF)), dict(logits=s[:, :0]),
               dict(val=v.clone().requires_grad_()), dict(weight=torch.ones(4, device="cuda", requires_grad=True))):
        for f in (topk_distill_loss, topk_distill_grad):
            with pytest.raises(lib.StesError):
                f(**{"logits": s, "idx": i, "val": v, **kw})
    for kw in (dict(accumulate=True), dict(out=s.half()), dict(out=s[:3]), dict(out=s), dict(out=torch.zeros(4, 1, device="cuda").expand(4, 7)),
               dict(out=torch.zeros(1, 7, device="cuda").expand(4, 7)), dict(out=torch.zeros(7, 4, device="cuda").t())):
        with pytest.raises((lib.StesError, RuntimeError)):
            topk_distill_grad(s, i, v, **kw)


# --------------------------------------------------------------------------------------------------------- together
def test_a_causal_head_is_distilled_over_ragged_videos():
    """Projection -> gated scan -> classes -> distillation from a teacher's top logits, as a student is trained on videos of different
    lengths: every gradient against float64 autograd of the same formulas."""
    from spot_amd.distill import topk_distill_loss
    from spot_amd.recurrence import gated_scan
    g = torch.Generator().manual_seed(0)
    B, T, D, H, V, k = 3, 150, 12, 16, 9, 4
    n = torch.tensor([150, 0, 77], dtype=torch.int32)
    x = torch.randn(B, T, D, generator=g)
    w1, w2, h0 = torch.randn(D, 2 * H, generator=g) * 0.5, torch.randn(H, V, generator=g), torch.randn(H, generator=g)
    val, idx = (torch.randn(B, T, V, generator=g) * 3).topk(k, 2)
    for b in range(B):
        idx[b, n[b]:] = -1
    leaves = [t.cuda().requires_grad_() for t in (w1, w2, h0)]
    h, _ = gated_scan(x.cuda() @ leaves[0], leaves[2], n.cuda())
    loss = topk_distill_loss(h @ leaves[1], idx.cuda(), val.cuda(), 2.0, denom=float(n.sum()))
    got = torch.autograd.grad(loss, leaves)
    ref = [t.double().requires_grad_() for t in (w1, w2, h0)]
    pre = x.double() @ ref[0]
    total = 0.0
    for b in range(B):
        s = ref[2]
        for t in range(int(n[b])):
            z = torch.sigmoid(pre[b, t, :H])
            s = (1 - z) * s + z * pre[b, t, H:]
            logq = torch.log_softmax(s @ ref[1] / 2.0, 0)
            p = torch.softmax(val[b, t].double() / 2.0, 0)
            total = total + (p * (p.log() - logq[idx[b, t]])).sum() * 4.0 / float(n.sum())
    want = torch.autograd.grad(total, ref)
    # fp32 throughout: sums of 227 frames' contributions, each good to some 100 u of its size (gates, softmax, products of 16 terms)
    assert abs(float(loss) - float(total)) <= 300 * SO.U * abs(float(total)) + 300 * SO.U
    for a, b in zip(got, want):
        assert float((a.double().cpu() - b).abs().max()) <= 2000 * SO.U * float(b.abs().max())
