"""A 1-rank communicator around the clip and the 4-bit policy's training: the
exchange's sums are identities."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import _lib, networks as nets
    from distributed_ddpg_amd.learner import FusedLearner, fill_synthetic, init_comm
    from distributed_ddpg_amd.replay_buffer import ReplayBuffer

NETS = {"small": (4, 1, 128, 200, 64), "large": (64, 16, 256, 256, 1024),
        "odd": (6, 3, 100, 60, 700)}


def make(size, comm, clip, dtype="fp32"):
    S, A, H1, H2, B = NETS[size]
    nets.reset_default_graph()
    actor = nets.ActorNetwork(S, A, 2.0, 1e-4, 1e-3, None, h1=H1, h2=H2)
    critic = nets.CriticNetwork(S, A, 1e-3, 1e-3, actor.get_num_trainable_vars(), None, h1=H1,
                                h2=H2)
    sess = nets.Session(device=0, batch_max=B, dtype=dtype, grad_clip=clip)
    actor.set_session(sess)
    critic.set_session(sess)
    sess.run(nets.global_variables_initializer(seed=7))
    if comm:
        init_comm(sess, 0, 1, single=True)
    return sess


def state(sess):
    return [sess.get_params(w, split=False) for w in range(10)]


@pytest.mark.parametrize("clip", [(float("inf"), float("inf")), (1e-3, 0.05)])
@pytest.mark.parametrize("size", sorted(NETS))
def test_a_clipped_step_has_the_same_bits(size, clip):
    S, A, H1, H2, B = NETS[size]
    got = []
    for comm in (False, True):
        sess = make(size, comm, clip)
        rb = ReplayBuffer(4 * B, 11)
        fill_synthetic(rb, S, A, 2 * B, scale=2.0, seed=3)
        learner = FusedLearner(sess, rb, B)
        for _ in range(3):
            learner.step()
        got.append(state(sess) + [np.array(sess.grad_norms())])
        sess.close()
    for a, b in zip(*got):
        assert np.array_equal(a, b), np.abs(a - b).max()


def trained(size, dtype, clip, steps):
    """train_mx's state without and with the communicator."""
    S, A, H1, H2, B = NETS[size]
    rng = np.random.default_rng(0)
    s, g = rng.standard_normal((B, S)).astype(np.float32), rng.standard_normal((B, A)).astype(np.float32)
    got = []
    for comm in (False, True):
        sess = make(size, comm, clip, dtype)
        for _ in range(steps):
            sess.actor.train_mx(s, g)
        got.append(state(sess))
        sess.close()
    return got


@pytest.mark.parametrize("clip", [None, (1e-3, None)])
@pytest.mark.parametrize("size", sorted(NETS))
def test_train_mx_has_the_same_bits(size, clip):
    for a, b in zip(*trained(size, "fp32", clip, 2)):
        assert np.array_equal(a, b), np.abs(a - b).max()


@pytest.mark.parametrize("size", sorted(NETS))
def test_train_mx_exchanges_as_a_bf16_context_does(size):
    """There a gradient is exchanged in bfloat16: the sum is rounded once."""
    a, b = (x[_lib.ACTOR_GRAD] for x in trained(size, "bf16", None, 1))
    assert np.array_equal(torch.from_numpy(a).bfloat16().float().numpy(), b)
