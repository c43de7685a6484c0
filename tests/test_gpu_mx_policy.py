"""The 4-bit policy (ddpg_actor_publish_mx / forward_mx / train_mx) against a
float64 actor whose hidden layer uses MXFP4 values (oracle/ops_oracle.py).

h1 is computed in float32 before it is quantised, so an h1 within float32's error
of a rounding border may take the other code than the float64 reference's.  That
error is a few 2^-24 against steps of 2^-1 to 2^-3 of the block's largest value, so
such an h1 is rare (about 1e-6 of them, times H1 a row): nine rows in ten are held
to float32's error, the rest to what a code more or less moves."""
import numpy as np
import pytest
import torch

from oracle import ops_oracle as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import _lib, networks as nets

SIZES = {"default": (4, 1, 128, 200, 256), "bench": (64, 16, 1024, 1024, 512),
         "odd": (5, 3, 100, 61, 130), "wide_state": (376, 17, 256, 192, 320)}


def make(size, dtype="fp32", clip=None):
    S, A, H1, H2, B = SIZES[size]
    nets.reset_default_graph()
    actor = nets.ActorNetwork(S, A, 2.0, 1e-3, 1e-3, None, h1=H1, h2=H2)
    critic = nets.CriticNetwork(S, A, 1e-3, 1e-3, actor.get_num_trainable_vars(), None, h1=H1,
                                h2=H2)
    sess = nets.Session(device=0, batch_max=B, dtype=dtype, grad_clip=clip)
    actor.set_session(sess)
    critic.set_session(sess)
    rng = np.random.default_rng(5)
    for which in (_lib.ACTOR, _lib.ACTOR_TARGET):
        sess.set_params(which, [rng.standard_normal(s).astype(np.float32) * (
            0.1 if len(s) == 1 else 1.0 / np.sqrt(s[0])) for s in actor.shapes()])
    for which in (_lib.CRITIC, _lib.CRITIC_TARGET):
        sess.set_params(which, [rng.standard_normal(s).astype(np.float32) * 0.1
                                for s in critic.shapes()])
    return sess, actor


def elu(x):
    return np.where(x < 0, np.expm1(x), x)


def forward(params, s):
    """(h1, quantised h1, quantised W2, h2, o) in float64, h1 rounded to float32
    before its quantisation."""
    W1, b1, W2, b2, W3 = [p.astype(np.float64) for p in params]
    h1 = elu(s.astype(np.float64) @ W1 + b1)
    h1q = O.mx_values(torch.from_numpy(h1.astype(np.float32))).numpy()
    w2q = O.mx_values(torch.from_numpy(np.ascontiguousarray(params[2].T))).numpy().T
    h2 = elu(h1q @ w2q + b2)
    return h1, h1q, w2q, h2, np.tanh(h2 @ W3)


def states(size, B=None):
    S, _, _, _, Bmax = SIZES[size]
    return np.random.default_rng(9).standard_normal((B or Bmax, S)).astype(np.float32)


@pytest.mark.parametrize("size", sorted(SIZES))
def test_predict(size):
    sess, actor = make(size)
    params = sess.get_params(_lib.ACTOR)
    with pytest.raises(_lib.DDPGError):
        actor.predict_mx(states(size, 1))
    actor.publish_mx()
    for B in (1, 7, 33, SIZES[size][4], SIZES[size][4] + 40):  # the last in pieces
        s = states(size, B)
        got = actor.predict_mx(s)
        want = 2.0 * forward(params, s)[4]
        assert got.shape == want.shape and got.dtype == np.float32
        err = np.abs(got - want).max(axis=1)
        # rows without an h1 next to a border: float32's error alone
        assert np.mean(err < 2e-5) > 0.9, err
        assert err.max() < 0.2
        # in the same batch class, a row does not depend on its neighbours
        assert np.array_equal(actor.predict_mx(s), got)
    assert actor.predict_mx(states(size)[:0]).shape == (0, SIZES[size][1])
    # near the full-precision policy, but not it
    full, four = actor.predict(states(size)), actor.predict_mx(states(size))
    d = np.abs(full - four)
    assert 0 < d.mean() < 0.25


def test_predict_bf16_context():
    """The first layer on bfloat16 operands (2^-9 each) moves some h1 across a
    border: the policy stays near the float32 context's."""
    sess, actor = make("wide_state", "bf16")
    actor.publish_mx()
    s = states("wide_state")
    want = 2.0 * forward(sess.get_params(_lib.ACTOR), s)[4]
    assert np.abs(actor.predict_mx(s) - want).mean() < 0.05


def test_the_worker_acts_on_it(tmp_path):
    from distributed_ddpg_amd import ddpg
    from distributed_ddpg_amd.parameters import Parameters
    opt = Parameters()
    opt.act_mx, opt.grad_clip = True, (0.5, 1.0)
    opt.batch_size, opt.rm_size, opt.hidden = 32, 1000, (32, 24)
    opt.summary_dir, opt.save_dir = str(tmp_path / "tb"), str(tmp_path / "model")
    nets.reset_default_graph()
    ddpg.run_worker(opt, 0, "synthetic", 2, 0)


def test_the_published_policy_stays():
    sess, actor = make("default")
    s = states("default", 20)
    actor.publish_mx()
    before = actor.predict_mx(s)
    g = np.ones((256, 1), np.float32)
    for _ in range(3):
        actor.train(states("default"), g)
        actor.train_mx(states("default"), g)
    assert np.array_equal(actor.predict_mx(s), before)
    actor.publish_mx()
    assert not np.array_equal(actor.predict_mx(s), before)
    actor.publish_mx(target=True)
    t = actor.predict_mx(s)
    want = 2.0 * forward(sess.get_params(_lib.ACTOR_TARGET), s)[4]
    assert np.mean(np.abs(t - want).max(axis=1) < 2e-5) > 0.9


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("size", sorted(SIZES))
def test_train_gradient(size, dtype):
    """The straight-through gradient of sum(a_gradient * -mu), as ActorNetwork.train
    forms it, against the float64 chain; bf16 contexts round the first layer's
    operands to bfloat16 (2^-9 each)."""
    sess, actor = make(size, dtype)
    S, A, H1, H2, B = SIZES[size]
    params = sess.get_params(_lib.ACTOR)
    W1, b1, W2, b2, W3 = [p.astype(np.float64) for p in params]
    s = states(size)
    ag = np.random.default_rng(1).standard_normal((B, A)).astype(np.float32)
    actor.train_mx(s, ag)
    h1, h1q, w2q, h2, o = forward(params, s)
    dz3 = -ag.astype(np.float64) * 2.0 * (1 - o * o)
    dz2 = (dz3 @ W3.T) * np.where(h2 < 0, h2 + 1, 1)
    dz1 = (dz2 @ w2q.T) * np.where(h1 < 0, h1 + 1, 1)
    want = [s.T.astype(np.float64) @ dz1, dz1.sum(0), h1q.T @ dz2, dz2.sum(0), h2.T @ dz3]
    tol = 2e-3 if dtype == "fp32" else 3e-2
    for g, w in zip(sess.get_params(_lib.ACTOR_GRAD), want):
        # a few h1 on the other side of a border move their share of a sum over B
        assert np.linalg.norm(g - w.reshape(g.shape)) < tol * np.linalg.norm(w), (
            g.shape, np.linalg.norm(g - w.reshape(g.shape)) / np.linalg.norm(w))
    # Adam's first step moved every parameter by about the learning rate
    p1 = sess.get_params(_lib.ACTOR)
    moved = np.abs(p1[2] - params[2])
    assert 0.9e-3 < np.median(moved[moved > 0]) < 1.1e-3


def test_train_is_clipped_and_repeats():
    s, g = states("default"), np.ones((256, 1), np.float32)
    a, actor = make("default")
    actor.train_mx(s, g)
    n = np.linalg.norm(a.get_params(_lib.ACTOR_GRAD, split=False).astype(np.float64))
    b, actor = make("default", clip=(n / 4, None))
    actor.train_mx(s, g)
    m = np.linalg.norm(b.get_params(_lib.ACTOR_GRAD, split=False).astype(np.float64))
    assert abs(b.grad_norms()[0] / n - 1) < 1e-6 and abs(m / (n / 4) - 1) < 1e-6
    c, actor = make("default", clip=(n / 4, None))
    actor.train_mx(s, g)
    assert np.array_equal(b.get_params(_lib.ACTOR, split=False),
                          c.get_params(_lib.ACTOR, split=False))


def test_refusals():
    sess, actor = make("odd")
    actor.publish_mx()
    with pytest.raises(ValueError):
        actor.train_mx(states("odd", 131), np.ones((131, 3), np.float32))
    with pytest.raises(ValueError):
        actor.train_mx(states("odd", 4)[:0], np.ones((0, 3), np.float32))
    with pytest.raises(ValueError):
        actor.predict_mx(np.zeros((4, 7), np.float32))
    out = np.zeros((200, 3), np.float32)
    s = np.zeros((200, 5), np.float32)
    assert _lib.lib.ddpg_actor_forward_mx(sess.ctx, _lib.fptr(s), 200, _lib.fptr(out)) == (
        _lib.DDPG_EINVAL)
