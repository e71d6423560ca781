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


def _refused(entry, cls, base, kw):
    import ctypes as C
    from spot_amd import lib
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where nothing can be launched")
    a = getattr(lib, cls)()
    for n, v in {**base, **kw}.items():
        setattr(a, n, v)
    return getattr(lib.lib(), entry)(C.byref(a), None) == -1 and b"share" in lib.lib().stes_last_error()


MB = 1 << 20


@pytest.mark.parametrize("kw", [dict(loss=MB + 40), dict(loss=2 * MB), dict(loss=3 * MB + 4), dict(weight=4 * MB), dict(loss=8 * MB, weight=8 * MB - 8), dict(loss=5 * MB + 12),
                                dict(stats=MB + 8), dict(stats=4 * MB), dict(stats=5 * MB + 4), dict(stats=2 * MB - 4), dict(ws=MB + 64), dict(ws=5 * MB), dict(stats=9 * MB, ws=9 * MB),
                                dict(ws=6 * MB - 8, loss=6 * MB), dict(zeros=MB - 65528), dict(zeros=5 * MB - 8), dict(upstream=5 * MB), dict(upstream=6 * MB), dict(zeros=6 * MB - 16)])
def test_distill_refuses_results_and_workspaces_that_share_memory(kw):
    base = dict(logits=MB, ld=600, f32=1, idx=2 * MB, ld_idx=4, val=3 * MB, ld_val=4, val_f32=1, M=30, V=600, k=4, temperature=1.0, denom=3.0, grad_scale=1.0,
                dlogits=5 * MB, ld_d=600, d_f32=1, loss=6 * MB, ws=7 * MB, ws_floats=1 << 20)
    if "weight" in kw and "loss" not in kw:
        kw = {**kw, "dlogits": 4 * MB - 8}
    if kw.get("stats") == 4 * MB:
        kw = {**kw, "weight": 4 * MB + 8}
    assert _refused("stes_distill", "DistillArgs", base, kw)


@pytest.mark.parametrize("kw", [dict(stats=5 * MB - 8), dict(stats=8 * MB, dlogits=8 * MB + 16), dict(upstream=5 * MB + 600)])
def test_distill_backward_refuses_a_gradient_over_what_it_reads(kw):
    base = dict(logits=MB, ld=600, f32=1, idx=2 * MB, ld_idx=4, val=3 * MB, ld_val=4, val_f32=1, M=30, V=600, k=4, temperature=1.0, denom=3.0, grad_scale=1.0,
                dlogits=5 * MB, ld_d=600, d_f32=1, stats=9 * MB)
    assert _refused("stes_distill_bwd", "DistillArgs", base, kw)


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("kw", [dict(ws=MB), dict(ws=2 * MB), dict(ws=3 * MB), dict(ws=4 * MB), dict(scrub=MB, scrub_bytes=16), dict(scrub=3 * MB + 16, scrub_bytes=16), dict(scrub=6 * MB + 16, scrub_bytes=16),
                                dict(scrub=4 * MB, scrub_bytes=32)])
def test_scan_refuses_workspaces_that_share_memory(kw, bwd):
    if bwd:
        base = dict(pre=MB, ld_pre=16, bs_pre=16000, dpre=2 * MB, ld_dpre=16, bs_dpre=16000, dh0=3 * MB, states=4 * MB, ws=6 * MB, ws_bytes=1 << 19, B=2, T=1000, H=8)
    else:
        base = dict(pre=MB, ld_pre=16, bs_pre=16000, h=2 * MB, ld_h=8, bs_h=8000, h_last=3 * MB, bs_hl=8, states=4 * MB, ws=6 * MB, ws_bytes=1 << 19, B=2, T=1000, H=8)
    assert _refused("stes_gated_scan_bwd" if bwd else "stes_gated_scan_fwd", "GatedScanArgs", base, kw)


def test_small_tensors_between_the_rows_of_a_gradient_do_not_share_memory(share):
    d = (MB, 4, 700, 0, 30, 1, 600)
    for at, n, want in ((600, 100, False), (600, 101, True), (599, 1, True), (1300, 1, False), (699, 1, False), (700, 1, True), (29 * 700 + 600, 10000, False)):
        assert share(d, (MB + 4 * at, 4, n, n, 1, 1, n)) is want


class _Engine:
    def __init__(self):
        self.flat, self.flat_grad, self.weights_dirty = torch.zeros(8), torch.zeros(8), False


class _Recorder:
    """The model side of DataParallelTrainer: keeps what the trainer hands to the step."""

    def __init__(self):
        self._model = torch.nn.Linear(1, 1)
        self._model.engine = _Engine()
        self.seen = []

    def train_step(self, frame, label, xy, lr, **kw):
        self.seen.append((kw["distill"], kw["ext_denoms"]))
        for lo, hi in ((4, 8), (0, 4)):
            kw["on_ready"](lo, hi)
        kw["after_backward"](self._model.engine)
        return torch.zeros(8)


def _denominator_worker(rank, world, port, q):
    import os
    import torch.distributed as dist
    from spot_amd.dp import DataParallelTrainer
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    m = _Recorder()
    t = DataParallelTrainer(m, dist)
    label = torch.zeros(3, 5, dtype=torch.int64)
    label[rank, 2] = 1
    given = {"idx": torch.zeros(3, 5, 2), "val": torch.zeros(3, 5, 2), "weight": 0.5}
    for d in (given, {**given, "denom": None}, {**given, "denom": 7.0}, None):
        m._model.engine.flat_grad.fill_(rank + 1.0)
        t.step(None, label, None, distill=d)
    q.put((rank, [None if d is None else (d["denom"], d["weight"]) for d, _ in m.seen], m.seen[0][1].tolist(), m._model.engine.flat_grad.tolist(), "denom" in given))
    dist.barrier()
    dist.destroy_process_group()


def test_distillation_denominator_counts_the_frames_of_all_ranks_gloo():
    from test_host_logic import _spawn_gloo
    for rank, seen, denoms, grad, touched in _spawn_gloo(_denominator_worker):
        assert seen == [(30.0, 0.5), (30.0, 0.5), (7.0, 0.5), None] and not touched
        assert denoms == [28 + 2 * 5.0, 2.0] and grad == [3.0] * 8


def test_distillation_denominator_of_one_process_is_the_callers():
    from spot_amd.dp import DataParallelTrainer
    m = _Recorder()
    m.train_step = lambda *a, **kw: m.seen.append(kw["distill"])
    d = {"idx": 0, "val": 0}
    DataParallelTrainer(m).step(None, torch.zeros(3, 5), None, distill=d)
    assert m.seen == [d]
