"""Entry points on no context (a session that was closed): an error code and a
message, for every ddpg_* call that takes one (no GPU needed)."""
import ctypes

import pytest

from distributed_ddpg_amd import _lib

# the calls whose first argument is a ddpg_ctx*; ddpg_destroy and ddpg_last_error
# take a null one, ddpg_create makes one
CTX = [n for n in open(_lib.__file__.replace("_lib.py", "../include/ddpg_hip.h")).read().split("\n")
       if n.startswith("int ddpg_") and "(ddpg_ctx* ctx" in n]
NAMES = sorted(n.split("(")[0].split()[1] for n in CTX)


def test_the_names_are_there():
    assert {"ddpg_sync", "ddpg_set_grad_clip", "ddpg_get_grad_norms", "ddpg_actor_publish_mx",
            "ddpg_actor_forward_mx", "ddpg_actor_train_mx", "ddpg_learner_step"} <= set(NAMES)


@pytest.mark.parametrize("name", NAMES)
def test_no_context_is_refused(name):
    fn = getattr(_lib.lib, name)
    args = [None] + [t(0) if t not in (ctypes.c_void_p,) and hasattr(t, "value") else None
                     for t in fn.argtypes[1:]]
    assert fn(*args) == _lib.DDPG_EINVAL
    assert b"context" in _lib.lib.ddpg_global_error()
