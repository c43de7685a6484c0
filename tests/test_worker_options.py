"""What the worker takes from an options object (no GPU: it stops where the device
context would open)."""
import pytest
import torch

from distributed_ddpg_amd import ddpg, networks as nets, replay_buffer
from distributed_ddpg_amd.parameters import Parameters


class Opened(Exception):
    pass


@pytest.fixture
def session(monkeypatch):
    seen = {}

    def open_session(*a, **kw):
        seen.update(kw)
        raise Opened

    monkeypatch.setattr(torch.cuda, "set_device", lambda device: None)
    monkeypatch.setattr(replay_buffer, "ReplayBuffer", lambda *a, **kw: None)
    monkeypatch.setattr(nets, "Session", open_session)
    nets.reset_default_graph()
    return seen


def run(opt):
    opt.batch_size, opt.rm_size = 32, 1000
    with pytest.raises(Opened):
        ddpg.run_worker(opt, 0, "synthetic", 1, 0)


def test_grad_clip_reaches_the_session(session):
    opt = Parameters()
    opt.grad_clip = (0.5, None)
    run(opt)
    assert session["grad_clip"] == (0.5, None)


def test_options_without_the_new_fields(session):
    """An options object of one's own, or one pickled earlier, has neither
    grad_clip nor act_mx: no clip, no 4-bit policy."""
    opt = Parameters()
    del opt.grad_clip, opt.act_mx
    run(opt)
    assert session["grad_clip"] is None
