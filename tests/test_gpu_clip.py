"""Gradient clipping by global norm inside the learner (ddpg_set_grad_clip):
the fused step on its small- and large-batch paths, the 1:1 train calls, graphs.

A clip that does not bind leaves every bit as it is without one; one that binds
gives the gradient times clip / norm (two float32 roundings: 2^-23 relative, the
norm another 2^-24) and the Adam update of that gradient."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import _lib, networks as nets
    from distributed_ddpg_amd.learner import FusedLearner, fill_synthetic
    from distributed_ddpg_amd.replay_buffer import ReplayBuffer

ALL = range(8)
NETS = {"small": (4, 1, 128, 200, 64), "large": (64, 16, 256, 256, 1024),
        "odd": (6, 3, 100, 60, 700)}


def make(size, dtype="fp32", clip=None):
    S, A, H1, H2, B = NETS[size]
    nets.reset_default_graph()
    actor = nets.ActorNetwork(S, A, 2.0, 1e-4, 1e-3, None, h1=H1, h2=H2)
    critic = nets.CriticNetwork(S, A, 1e-3, 1e-3, actor.get_num_trainable_vars(), None, h1=H1,
                                h2=H2)
    sess = nets.Session(device=0, batch_max=B, dtype=dtype, grad_clip=clip)
    actor.set_session(sess)
    critic.set_session(sess)
    sess.run(nets.global_variables_initializer(seed=7))
    rb = ReplayBuffer(4 * B, 11)
    fill_synthetic(rb, S, A, 2 * B, scale=2.0, seed=3)
    return sess, FusedLearner(sess, rb, B)


def norm(sess, which):
    g = sess.get_params(which, split=False).astype(np.float64)
    return float(np.sqrt((g * g).sum()))


def state(sess):
    return [sess.get_params(w, split=False) for w in ALL]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", sorted(NETS))
def test_a_clip_that_does_not_bind_changes_nothing(size, dtype):
    plain, a = make(size, dtype)
    inf, b = make(size, dtype, math.inf)
    wide, c = make(size, dtype, (1e6, None))
    for _ in range(4):
        sa, sb, sc = a.step(stats=True), b.step(stats=True), c.step(stats=True)
        assert sa == sb == sc
    for x, y, z in zip(state(plain), state(inf), state(wide)):
        assert np.array_equal(x, y) and np.array_equal(x, z)
    na, nc = inf.grad_norms()
    assert abs(na / norm(inf, _lib.ACTOR_GRAD) - 1) < 2.0 ** -22
    assert abs(nc / norm(inf, _lib.CRITIC_GRAD) - 1) < 2.0 ** -22
    na, nc = wide.grad_norms()
    assert na > 0 and math.isnan(nc)
    assert a.read_stats() == b.read_stats() == c.read_stats()
    with pytest.raises(_lib.DDPGError):
        plain.grad_norms()


@pytest.mark.parametrize("net", ["actor", "critic"])
@pytest.mark.parametrize("size", sorted(NETS))
def test_a_binding_clip_scales_the_gradient(size, net):
    """One step from equal state: the clipped network's gradient, moments and
    parameters.  (With the critic unclipped, the actor's gradient is the same.)"""
    grad, theta, m, v = ((_lib.ACTOR_GRAD, _lib.ACTOR, _lib.ACTOR_ADAM_M, _lib.ACTOR_ADAM_V)
                         if net == "actor" else
                         (_lib.CRITIC_GRAD, _lib.CRITIC, _lib.CRITIC_ADAM_M, _lib.CRITIC_ADAM_V))
    lr = 1e-4 if net == "actor" else 1e-3
    plain, a = make(size)
    p0 = plain.get_params(theta, split=False).astype(np.float64)
    a.step()
    g = plain.get_params(grad, split=False).astype(np.float64)
    n = norm(plain, grad)
    clip = np.float32(0.25 * n)
    sess, b = make(size, clip=(clip, None) if net == "actor" else (None, clip))
    b.step()
    got = sess.get_params(grad, split=False)
    want = g * (float(clip) / n)
    assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -21 + 1e-44)
    seen = sess.grad_norms()[0 if net == "actor" else 1]
    assert abs(seen / n - 1) < 2.0 ** -22
    # ApplyAdam's first step on the clipped gradient
    gc = got.astype(np.float64)
    assert np.allclose(sess.get_params(m, split=False), gc * 0.1, rtol=1e-6, atol=1e-44)
    assert np.allclose(sess.get_params(v, split=False), gc * gc * 0.001, rtol=1e-4, atol=1e-40)
    alpha = lr * math.sqrt(1 - 0.999) / (1 - 0.9)
    step = 0.1 * gc * alpha / (np.sqrt(0.001 * gc * gc) + 1e-8)
    p1 = sess.get_params(theta, split=False)
    assert np.all(np.abs(p1 - (p0 - step)) <= np.abs(p0) * 2.0 ** -23 + np.abs(step) * 1e-3 + 1e-12)


def test_the_clip_can_change_between_graph_steps():
    sess, a = make("large")
    a.step()
    n = norm(sess, _lib.CRITIC_GRAD)
    sess.set_grad_clip(critic=0.1 * n)
    for i in range(4):  # both graph slots
        a.step()
        assert abs(norm(sess, _lib.CRITIC_GRAD) / (0.1 * n) - 1) < 1e-5 or (
            sess.grad_norms()[1] < 0.1 * n)
    sess.set_grad_clip(critic=0.01 * n)
    for i in range(3):
        a.step()
        assert norm(sess, _lib.CRITIC_GRAD) <= 0.01 * n * 1.00001
        assert math.isnan(sess.grad_norms()[0])
    sess.set_grad_clip()
    a.step()
    assert norm(sess, _lib.CRITIC_GRAD) > 0.01 * n
    assert all(math.isnan(x) for x in sess.grad_norms())


@pytest.mark.parametrize("size", ["small", "large"])
def test_train_calls_are_clipped(size):
    S, A, H1, H2, B = NETS[size]
    rng = np.random.default_rng(0)
    s = rng.standard_normal((B, S)).astype(np.float32)
    act = rng.uniform(-1, 1, (B, A)).astype(np.float32)
    y = rng.standard_normal((B, 1)).astype(np.float32)
    plain, _ = make(size)
    plain.critic.train(s, act, y)
    plain.actor.train(s, act)
    n = [norm(plain, _lib.ACTOR_GRAD), norm(plain, _lib.CRITIC_GRAD)]
    sess, _ = make(size, clip=(n[0] / 3, n[1] / 5))
    sess.critic.train(s, act, y)
    sess.actor.train(s, act)
    for g, x, k in ((_lib.ACTOR_GRAD, n[0], 3), (_lib.CRITIC_GRAD, n[1], 5)):
        assert abs(norm(sess, g) / (x / k) - 1) < 1e-5
        want = plain.get_params(g, split=False) / k
        got = sess.get_params(g, split=False)
        assert np.allclose(got, want, rtol=1e-5, atol=1e-7 * np.abs(want).max())


def test_refusals():
    for bad in (0, -1.0, math.nan, (1.0,), (1.0, -2.0), (1.0, 2.0, 3.0)):
        with pytest.raises(ValueError):
            make("small", clip=bad)
    sess, _ = make("small")
    for x in (-1.0, math.nan):
        rc = _lib.lib.ddpg_set_grad_clip(sess.ctx, x, 1.0)
        assert rc == _lib.DDPG_EINVAL


@pytest.mark.parametrize("size", ["small", "large"])
def test_the_clip_follows_the_exchange(size):
    """A 1-rank communicator runs the data-parallel order (gradient, sum, norm,
    Adam); its sums are identities, so every bit is the communicator-less step's."""
    from distributed_ddpg_amd.learner import init_comm
    one, a = make(size, clip=(1e-3, 0.05))
    two, b = make(size, clip=(1e-3, 0.05))
    init_comm(two, 0, 1, single=True)
    # (a communicator's small step reads the summed gradient back in its Adam
    # launch, as a clipped step does; the large one adds its slabs the same way)
    for _ in range(3):
        a.step()
        b.step()
    for x, y in zip(state(one), state(two)):
        assert np.allclose(x, y, rtol=1e-5, atol=1e-8 + 1e-6 * np.abs(x).max())
    assert np.allclose(one.grad_norms(), two.grad_norms(), rtol=1e-5)
    two.close()
