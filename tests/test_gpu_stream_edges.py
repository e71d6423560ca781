"""Frame streams and training against a teacher where the call could go wrong: states that do not fit, heads and backbones that look
ahead, clips trained backwards in time."""
import numpy as np
import pytest
import torch

from test_gpu_stream_distill import _batch, _frames, _model, fixed_order, rel  # noqa: F401

pytestmark = pytest.mark.gpu


def test_stream_states_that_do_not_fit_are_refused_before_any_moves_on():
    from spot_amd import lib
    m = _model()
    x = _frames(4)[None].cuda()
    wrong = (lambda s: s.cpu(), lambda s: s[0], lambda s: s[None], lambda s: s.expand(2, -1), lambda s: None)
    for change in wrong:
        for at in (0, 2):
            state = m.new_stream()
            state[at] = change(state[at])
            old = [None if s is None else s.clone() for s in state]
            with pytest.raises(lib.StesError):
                m.predict_stream(x, state)
            assert all(a is b or torch.equal(a, b) for a, b in zip(state, old))
    for state in (None, 3, m.new_stream()[0]):
        with pytest.raises(lib.StesError):
            m.predict_stream(x, state)
