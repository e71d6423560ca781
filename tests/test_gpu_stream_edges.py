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


def test_streams_refuse_a_backbone_that_looks_ahead():
    """Channel attention gates a clip's frames by their mean over the whole clip: a frame's features depend on later frames, and on the
    cut into clips."""
    from spot_amd.e2e import E2EModel
    from spot_amd.infer import run_inference
    m = E2EModel(7, "rny008", "mingru", clip_len=4, modality="rgb", device="cuda", predict_location=True, use_channel_attention=True, verbose=False)
    with pytest.raises(NotImplementedError):
        m.new_stream()
    state = [h.detach().cuda().float().expand(1, -1).clone() for h in m._model._pred_fine.h0]
    with pytest.raises(NotImplementedError):
        m.predict_stream(_frames(4)[None].cuda(), state)
    with pytest.raises(NotImplementedError):
        run_inference(m, _frames(8), ["c%d" % i for i in range(1, 7)], 4, carry_state=True)
