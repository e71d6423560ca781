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


@pytest.mark.parametrize("tarch,teacher", [("mingru", True), ("mingru", False), ("", True)])
def test_fused_step_of_a_time_backward_model_matches_the_autograd_loop(fixed_order, tarch, teacher):  # noqa: F811
    """The fused step turns the clips round in time as the module's forward does, and labels, locations and the teacher's lists with them."""
    import torch.nn.functional as F
    from spot_amd.distill import topk_distill_loss
    from spot_amd.e2e import E2EModel

    def model():
        torch.manual_seed(5)
        return E2EModel(7, "rny008_tsm", tarch, clip_len=4, modality="rgb", device="cuda", predict_location=True, time_backward=True, verbose=False)
    frame, label, xy, idx, val = _batch()
    fw = torch.rand(2, 4, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    given = [t.clone() for t in (frame, label, xy, idx, val, fw)]
    m = model()
    state = m._model.state_dict()
    distill = {"idx": idx, "val": val, "temperature": 2.0, "weight": 0.7, "frame_weight": fw} if teacher else None
    out = m.train_step(frame, label, xy, 0.0, optimizer_step=False, distill=distill).clone()
    assert all(torch.equal(a, b) for a, b in zip(given, (frame, label, xy, idx, val, fw)))
    eng = m._model.engine
    got = {n: eng.grad(p).clone() for n, p in m._model.named_parameters() if n.startswith("_pred") and p.requires_grad}
    m2 = model()
    m2._model.load_state_dict(state)
    m2._model.train()
    d = m2._model(frame)
    cls = F.cross_entropy(d["im_feat"].reshape(-1, 7), label.reshape(-1), weight=torch.tensor([1.0] + [5.0] * 6).cuda())
    mask = (label != 0).float().reshape(-1)
    loc = (F.l1_loss(d["loc_feat"].reshape(-1, 2).sigmoid(), xy.reshape(-1, 2), reduction="none").sum(1) * mask).sum() / (mask.sum() + 1e-6)
    kd = topk_distill_loss(d["im_feat"], idx, val, 2.0, fw) if teacher else 0.0 * cls
    (cls + loc + 0.7 * kd).backward()
    np.testing.assert_allclose(out[:3].cpu().numpy(), [float(cls + loc + 0.7 * kd), float(cls), float(loc)], rtol=1e-4)
    for n, p in m2._model.named_parameters():
        if n in got:
            assert rel(got[n], p.grad) < 2e-2, n          # (class gradients rounded to bf16 once there, twice here)
