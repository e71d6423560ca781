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
