"""Forward-mode duals (no GPU needed: the check comes before the first device
call).  An operator without a formula for the tangent refuses it, also where grad
mode is off, which does not switch forward mode off."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from distributed_ddpg_amd import ops

CALLS = {"norm": lambda d, t: ops.global_norm([d, t]),
         "clip": lambda d, t: ops.clip_by_global_norm([d], 1.0),
         "clip in place": lambda d, t: ops.clip_by_global_norm([d], 1.0, inplace=True),
         "quantise": lambda d, t: ops.mx_quantize(d)}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call", sorted(CALLS))
def test_a_dual_is_refused(call, grad):
    t = torch.ones(4, 4)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        d = fw.make_dual(t, torch.ones(4, 4))
        with pytest.raises(ValueError, match="tangent"):
            CALLS[call](d, t)
        # without its tangent it is a tensor like any other (here: of the wrong device)
        with pytest.raises(ValueError, match="GPU"):
            CALLS[call](d.detach(), t)
    with pytest.raises(ValueError, match="GPU"):
        CALLS[call](t, t)
