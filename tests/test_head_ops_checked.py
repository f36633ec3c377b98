"""The norm, the e4m3 products and the clipped steps on the CPU: calls that used to be
answered wrongly or forgotten, each with what it has to give."""

import pytest
import torch

from active_learning_amd.ops.optim import FusedSGD


def _params(sizes):
    ps = [torch.nn.Parameter(torch.randn(s)) for s in sizes]
    for p in ps:
        p.grad = torch.randn_like(p)
    return ps


@pytest.fixture
def capturing(monkeypatch):
    """A switch that makes torch say that the stream is being captured."""
    state = {"on": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["on"])
    return lambda on: state.update(on=on)


@pytest.mark.parametrize("bound", [None, 0.5])
def test_momentum_cannot_come_after_the_capture(capturing, bound):
    """A step that is captured without momentum has no buffers for it."""
    opt = FusedSGD(_params([(3, 4)]), lr=0.1, max_grad_norm=bound)
    opt.enable_device_hyper("cpu")
    opt.step()
    capturing(True)
    opt.step()
    capturing(False)
    opt.param_groups[0]["lr"] = 0.05
    opt.sync_hyper()
    opt.param_groups[0]["momentum"] = 0.9
    with pytest.raises(ValueError, match="captured without momentum"):
        opt.sync_hyper()
    assert opt._hyper_dev[1] == 0
    # with buffers at the capture it may come and go
    opt = FusedSGD(_params([(3, 4)]), lr=0.1, momentum=0.9, max_grad_norm=bound)
    opt.enable_device_hyper("cpu")
    opt.step()
    opt.param_groups[0]["momentum"] = 0.0
    opt.sync_hyper()
    capturing(True)
    opt.step()
    capturing(False)
    opt.param_groups[0]["momentum"] = 0.9
    opt.sync_hyper()
    assert abs(opt._hyper_dev[1] - 0.9) < 1e-6
