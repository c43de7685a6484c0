"""The worker's use of Parameters.act_mx and grad_clip: what it calls, counted."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import _lib, networks as nets


absent = object()


def run(tmp_path, monkeypatch, episodes=3, **fields):
    """run_worker with these options: how often it called each, and the clip its
    session had."""
    from distributed_ddpg_amd import ddpg
    from distributed_ddpg_amd.parameters import Parameters
    calls = dict.fromkeys(("publish_mx", "predict_mx", "predict"), 0)
    seen = {}

    def counted(name):
        plain = getattr(nets.ActorNetwork, name)

        def call(self, *a, **kw):
            calls[name] += 1
            return plain(self, *a, **kw)
        return call

    for name in calls:
        monkeypatch.setattr(nets.ActorNetwork, name, counted(name))
    close = nets.Session.close

    def closing(sess):
        if sess.ctx:  # not the second time, by __del__
            try:
                seen["norms"] = sess.grad_norms()
            except _lib.DDPGError:
                seen["norms"] = None
        close(sess)

    monkeypatch.setattr(nets.Session, "close", closing)
    opt = Parameters()
    opt.batch_size, opt.rm_size, opt.hidden = 8, 1000, (32, 24)
    opt.summary_dir, opt.save_dir = str(tmp_path / "tb"), str(tmp_path / "model")
    for k, v in fields.items():
        setattr(opt, k, v)
        if v is absent:
            delattr(opt, k)
    env = {}
    make_env = ddpg.make_env

    def counting(*a):
        e = make_env(*a)
        step = e.step

        def one(x):
            env["steps"] = env.get("steps", 0) + 1
            return step(x)
        e.step = one
        return e

    monkeypatch.setattr(ddpg, "make_env", counting)
    nets.reset_default_graph()
    ddpg.run_worker(opt, 0, "synthetic", episodes, 0)
    return calls, env["steps"], seen


def test_it_acts_on_the_published_policy(tmp_path, monkeypatch):
    calls, steps, seen = run(tmp_path, monkeypatch, act_mx=True, grad_clip=(0.5, 1.0))
    assert steps > 8  # the replay held a batch: updates ran
    assert calls == {"publish_mx": 3, "predict_mx": steps, "predict": 0}
    assert seen["norms"] is not None and all(n > 0 for n in seen["norms"])


@pytest.mark.parametrize("fields", [{}, {"act_mx": absent, "grad_clip": absent}])
def test_it_acts_in_full_precision_without(tmp_path, monkeypatch, fields):
    calls, steps, seen = run(tmp_path, monkeypatch, **fields)
    assert calls == {"publish_mx": 0, "predict_mx": 0, "predict": steps}
    assert seen["norms"] is None
