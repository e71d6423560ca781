"""The 64-bit restatements of the gated scan and of the top-logits distillation (oracle/sequence_oracle.py) against torch's
autograd in float64 and against differences; the refusals of the Python entry points and of the C-ABI (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO


def _torch_scan(pre, h0, lengths, reverse):
    B, T, W = pre.shape
    H = W // 2
    hs, lasts = [], []
    for b in range(B):
        n = T if lengths is None else int(min(max(int(lengths[b]), 0), T))
        x, rows = h0[b], [torch.zeros(H, dtype=torch.float64)] * T
        for t in (range(n - 1, -1, -1) if reverse else range(n)):
            z = torch.sigmoid(pre[b, t, :H])
            x = (1 - z) * x + z * pre[b, t, H:]
            rows[t] = x
        hs.append(torch.stack(rows) if T else torch.zeros(0, H, dtype=torch.float64))
        lasts.append(x)
    return torch.stack(hs), torch.stack(lasts)


@pytest.mark.parametrize("T,lengths,reverse", [(1, None, False), (9, None, True), (7, [0, 3, 7], False), (7, [7, -2, 99], True), (0, None, False)])
def test_scan_oracle_against_autograd_and_differences(T, lengths, reverse):
    rng = np.random.default_rng(T + 3)
    B, H = 3, 4
    pre, h0 = rng.normal(size=(B, T, 2 * H)) * 2, rng.normal(size=(B, H))
    dh, dlast = rng.normal(size=(B, T, H)), rng.normal(size=(B, H))
    got = SO.gated_scan(pre, h0, lengths, reverse, dh, dlast, need_grad=True)
    tp, t0 = torch.tensor(pre, requires_grad=True), torch.tensor(h0, requires_grad=True)
    h, last = _torch_scan(tp, t0, lengths, reverse)
    np.testing.assert_allclose(got["h"], h.detach(), rtol=0, atol=1e-13)
    np.testing.assert_allclose(got["last"], last.detach(), rtol=0, atol=1e-13)
    ((h * torch.tensor(dh)).sum() + (last * torch.tensor(dlast)).sum()).backward()
    if T:
        np.testing.assert_allclose(got["dpre"], tp.grad, rtol=0, atol=1e-12)
    np.testing.assert_allclose(got["dh0"], t0.grad, rtol=0, atol=1e-12)

    def value(p, s):
        r = SO.gated_scan(p, s, lengths, reverse)
        return (r["h"] * dh).sum() + (r["last"] * dlast).sum()
    vp, v0, e = rng.normal(size=pre.shape), rng.normal(size=h0.shape), 1e-5
    slope = (value(pre + e * vp, h0 + e * v0) - value(pre - e * vp, h0 - e * v0)) / (2 * e)
    # central differences: O(e^2) = 1e-10 of a third derivative of order 10, and 1e-16 / e = 1e-11 of rounding
    np.testing.assert_allclose((got["dpre"] * vp).sum() + (got["dh0"] * v0).sum(), slope, rtol=0, atol=1e-6)


@pytest.mark.parametrize("V,k,tau,weighted", [(7, 4, 1.0, True), (2, 2, 3.0, False), (40, 1, 0.5, True)])
def test_distill_oracle_against_autograd_and_differences(V, k, tau, weighted):
    rng = np.random.default_rng(V)
    M = 5
    x, val = rng.normal(size=(M, V)) * 3, rng.normal(size=(M, k)) * 3
    idx = np.stack([rng.permutation(V)[:k] for _ in range(M)])
    idx[1] = -1                                                          # a row that lists nothing
    if k > 1:
        idx[2, 0] = -1
        idx[3, 1] = idx[3, 0]                                            # a class listed twice
    w = rng.uniform(0.5, 2, size=M) if weighted else None
    got = SO.topk_distill(x, idx, val, tau, w, denom=3.0)
    t = torch.tensor(x, requires_grad=True)
    loss = 0.0
    for m in range(M):
        on = idx[m] >= 0
        if not on.any():
            continue
        p = torch.zeros(V, dtype=torch.float64).index_add(0, torch.tensor(idx[m][on]), torch.softmax(torch.tensor(val[m][on]) / tau, 0))
        kl = torch.nn.functional.kl_div(torch.log_softmax(t[m] / tau, 0), p, reduction="sum")
        loss = loss + (1.0 if w is None else w[m]) * kl * tau ** 2 / 3.0
    loss.backward()
    np.testing.assert_allclose(got["loss"], loss.detach(), rtol=1e-13)
    np.testing.assert_allclose(got["dlogits"], t.grad, rtol=0, atol=1e-13)
    v, e = rng.normal(size=x.shape), 1e-5
    slope = (SO.topk_distill(x + e * v, idx, val, tau, w, 3.0)["loss"] - SO.topk_distill(x - e * v, idx, val, tau, w, 3.0)["loss"]) / (2 * e)
    np.testing.assert_allclose((got["dlogits"] * v).sum(), slope, rtol=0, atol=1e-7)


def test_python_entry_points_refuse_host_tensors_and_wrong_types():
    from spot_amd import lib
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    from spot_amd.recurrence import gated_scan
    for bad in (torch.zeros(2, 3, 8), torch.zeros(3, 8), torch.zeros(2, 3, 8, dtype=torch.float16), None):
        with pytest.raises(lib.StesError):
            gated_scan(bad)
    i, v = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    for f in (topk_distill_loss, topk_distill_grad):
        for x in (torch.zeros(4, 7), torch.zeros(4, 7, dtype=torch.float64)):
            with pytest.raises(lib.StesError):
                f(x, i, v)


def _refused(entry, a):
    from spot_amd import lib
    rc = getattr(lib.lib(), entry)(None if a is None else C.byref(a), None)
    assert rc < 0 and lib.lib().stes_last_error(), (entry, rc)
    return rc


def _scan_args(**kw):
    from spot_amd import lib
    a = lib.GatedScanArgs()
    base = dict(pre=1 << 20, ld_pre=16, bs_pre=64, h=2 << 20, ld_h=8, bs_h=32, h_last=3 << 20, bs_hl=8, states=4 << 20, dpre=5 << 20, ld_dpre=16, bs_dpre=64,
                ws=256, ws_bytes=1 << 40, B=2, T=4, H=8)
    for n, v in {**base, **kw}.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [dict(B=-1), dict(T=-1), dict(H=-1), dict(f32=2), dict(pre=None), dict(h=None), dict(ld_pre=15), dict(ld_h=7), dict(bs_h=31), dict(bs_h=0),
                                dict(bs_hl=7), dict(h0=512, bs_h0=3), dict(h0=3 << 20, bs_h0=0), dict(h0=3 << 20, bs_h0=9),
                                dict(h0=(3 << 20) + 4, bs_h0=8), dict(h0=(2 << 20) + 16, bs_h0=8), dict(h=(1 << 20) + 16), dict(h=(1 << 20) - 2), dict(h=(1 << 20) + 32, ld_h=16, bs_h=64, B=1, T=3, ld_pre=23),
                                dict(h_last=(1 << 20) + 200), dict(h_last=(2 << 20) + 8), dict(states=(2 << 20)), dict(lengths=(3 << 20) + 4), dict(lengths=(2 << 20) - 4),
                                dict(pre=1 << 20, h=(1 << 20) + 32, ld_pre=23, bs_pre=92, ld_h=23, bs_h=92), dict(pre=1 << 20, h=(1 << 20) + 34, ld_pre=24, bs_pre=96, ld_h=24, bs_h=96),
                                dict(pre=1 << 20, h=(1 << 20) + 32, ld_pre=24, bs_pre=94, ld_h=24, bs_h=94), dict(scrub=256, scrub_bytes=16), dict(T=1000, bs_pre=16000, bs_h=8000, ws=264),
                                dict(T=1000, bs_pre=16000, bs_h=8000, ws_bytes=16), dict(T=1000, bs_pre=16000, bs_h=8000, scrub=256, scrub_bytes=8),
                                dict(B=70000000, H=1 << 20), dict(B=1 << 23, T=1, H=64, ld_pre=128, bs_pre=128, bs_h=64, ld_h=64, bs_hl=64)])
def test_scan_forward_refuses(kw):
    _refused("stes_gated_scan_fwd", _scan_args(**kw))


@pytest.mark.parametrize("kw", [dict(states=None), dict(dpre=None), dict(ld_dpre=15), dict(bs_dpre=63), dict(dh=256, ld_dh=7), dict(dh0_sum=256), dict(scrub=256, scrub_bytes=16),
                                dict(dpre=1 << 20), dict(dpre=(1 << 20) + 250), dict(dh=(5 << 20) + 16, ld_dh=8, bs_dh=32), dict(dh0=(4 << 20)), dict(dh0=(5 << 20) + 4),
                                dict(dh0=6 << 20, dh0_sum=(6 << 20) + 32), dict(dh0=6 << 20, dh_last=6 << 20, bs_dhl=8)])
def test_scan_backward_refuses(kw):
    _refused("stes_gated_scan_bwd", _scan_args(**kw))


def _distill_args(**kw):
    from spot_amd import lib
    a = lib.DistillArgs()
    base = dict(logits=1 << 20, ld=7, idx=2 << 20, ld_idx=4, val=3 << 20, ld_val=4, M=3, V=7, k=4, temperature=1.0, denom=3.0, grad_scale=1.0, loss=256,
                ws=256, ws_floats=1 << 40)
    for n, v in {**base, **kw}.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [dict(M=-1), dict(V=0), dict(k=0), dict(k=65, ld_idx=65, ld_val=65), dict(temperature=0.0), dict(temperature=-1.0),
                                dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-7), dict(temperature=2e6), dict(denom=0.0), dict(denom=float("nan")),
                                dict(logits=None), dict(idx=None), dict(val=None), dict(loss=None), dict(ld=6), dict(ld_idx=3), dict(ld_val=3),
                                dict(dlogits=512, ld_d=6), dict(dlogits=1 << 20, ld_d=7), dict(dlogits=(1 << 20) + 40, ld_d=7), dict(dlogits=(1 << 20) - 2, ld_d=9), dict(dlogits=(2 << 20) + 47, ld_d=7),
                                dict(dlogits=3 << 20, ld_d=7), dict(weight=(4 << 20) + 20, dlogits=4 << 20, ld_d=7), dict(ld=13, dlogits=(1 << 20) + 14, ld_d=13), dict(M=1 << 22, V=1000, ld=1000),
                                dict(M=1000, V=1000, ld=1000, ws_floats=999), dict(M=100, V=1000, ld=1000, ws=None), dict(M=3000, ws_floats=46), dict(M=100, V=1000, ld=1000, zeros=1 << 25, ws=None, stats=None, loss=None), dict(zeros=(1 << 25) + 4),
                                dict(M=4097, V=1000, ld=1000, zeros=1 << 25, ws_floats=4096)])
def test_distill_refuses(kw):
    _refused("stes_distill", _distill_args(**kw))


def test_distill_backward_and_null_refuse():
    _refused("stes_distill_bwd", _distill_args(dlogits=512, ld_d=7))
    _refused("stes_distill_bwd", _distill_args(stats=512))
    for e in ("stes_distill", "stes_distill_bwd", "stes_gated_scan_fwd", "stes_gated_scan_bwd"):
        _refused(e, None)
