"""The sequence operators' host side where no GPU is needed: what refuses to be recorded, memory that a call shares, sizes at the end of
their types, the data-parallel denominators."""
import pytest
import torch


def _calls():
    from spot_amd.distill import topk_distill_grad, topk_distill_loss
    from spot_amd.recurrence import gated_scan
    i, v = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    return [(torch.zeros(2, 3, 8), lambda t: gated_scan(t)[0]), (torch.zeros(4, 7), lambda t: topk_distill_loss(t, i, v)),
            (torch.zeros(4, 7), lambda t: topk_distill_grad(t, i, v)[1])]


def test_tracing_is_refused():
    """A trace would hold the allocation of a result and not the call that writes it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from spot_amd import lib
    for x, f in _calls():
        for check in (True, False):
            with pytest.raises(lib.StesError, match="trace"):
                torch.jit.trace(f, (x,), check_trace=check)
        for kw in (dict(), dict(tracing_mode="fake"), dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
            with pytest.raises(lib.StesError, match="trace"):
                make_fx(f, **kw)(x)
        with pytest.raises(lib.StesError) as e:            # (and the refusal of a host tensor is another one)
            f(x)
        assert "trace" not in str(e.value)


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    """stes_share (csrc/stes_share.h) as a function of two layouts (address, element bytes, ld, bs, T, B, width)."""
    import ctypes as C
    import os
    import subprocess
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    d = tmp_path_factory.mktemp("share")
    (d / "s.cpp").write_text('#include "%s"\nextern "C" int share(const long long* q) {\n'
                             '    auto r = [](const long long* v) { return StesRows{(const void*)v[0], (int)v[1], v[2], v[3], v[4], v[5], v[6]}; };\n'
                             '    return stes_share(r(q), r(q + 7));\n}\n' % os.path.join(here, "spot_amd", "csrc", "stes_share.h"))
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(d / "s.cpp"), "-o", str(d / "s.so")])
    fn = C.CDLL(str(d / "s.so")).share
    return lambda a, b: bool(fn((C.c_longlong * 14)(*a, *b)))


def _elements(p, es, ld, bs, T, B, width):
    return {p // es + t * ld + b * bs + v for t in range(T) for b in range(B) for v in range(width)}


@pytest.mark.parametrize("B", [3, 33, 34, 100, 1000])
@pytest.mark.parametrize("T", [1, 2, 7, 300])
def test_columns_of_one_buffer_do_not_share_memory(share, B, T):
    """pre in the first 2H of 3H columns and h in the last, frames or sequences outermost; one column to the left they share."""
    H, p = 8, 1 << 20
    for ld, bs in ((3 * H, 3 * H * T), (3 * H * B, 3 * H)):
        pre = (p, 4, ld, bs, T, B, 2 * H)
        for off, want in ((2 * H, False), (2 * H - 1, True), (0, True), (H, True)):
            h = (p + 4 * off, 4, ld, bs, T, B, H)
            assert share(pre, h) is want and share(h, pre) is want
        late = (p + 4 * ld * T, 4, ld, bs, T, B, H)                      # the frames behind (frames outermost: behind all)
        assert share(pre, late) is bool(_elements(*pre) & _elements(*late))


def test_shared_memory_against_sets_of_elements(share):
    """Random layouts of equal strides: never missed, and refused wrongly only where a batch's sequences lie across one another."""
    import random
    rng = random.Random(5)
    wrong = 0
    for _ in range(20000):
        T, B, w1, w2 = rng.randint(1, 6), rng.randint(1, 6), rng.randint(1, 5), rng.randint(1, 5)
        inner = rng.randint(max(w1, w2), 12)
        outer = inner * max(T, B) + rng.randint(0, 5)
        ld, bs = (inner, outer) if rng.random() < 0.5 else (outer, inner)
        a = (4096, 4, ld, bs, T, B, w1)
        b = (4096 + 4 * rng.randint(-80, 80), 4, ld, bs, rng.choice((1, T)), rng.choice((1, B)), w2)
        truth = bool(_elements(*a) & _elements(*b))
        assert not truth or share(a, b), (a, b)
        wrong += share(a, b) and not truth
    assert wrong == 0


@pytest.mark.parametrize("T", [2**31 - 1, 2**31 - 200, 2**31 - 255, 2**31 - 511])
def test_scan_refuses_lengths_next_to_the_end_of_32_bits(T):
    import ctypes as C
    from spot_amd import lib
    L = lib.lib()
    assert L.stes_gated_scan_ws_bytes(1, T, 1) == 256 + 16 * 64 * (-(-T // 256))
    a = lib.GatedScanArgs()
    for n, v in dict(pre=1 << 40, ld_pre=2, bs_pre=2 * T, h=2 << 40, ld_h=1, bs_h=T, h_last=3 << 40, bs_hl=1, states=4 << 40, dpre=5 << 40, ld_dpre=2, bs_dpre=2 * T,
                     ws=6 << 40, ws_bytes=1 << 38, B=1, T=T, H=1).items():
        setattr(a, n, v)
    for e in (L.stes_gated_scan_fwd, L.stes_gated_scan_bwd):
        assert e(C.byref(a), None) == lib.ERR_UNSUPPORTED
