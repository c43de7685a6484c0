"""Tensor operators (distributed_ddpg_amd/ops.py) on the GPU, at the edges of what
a call may bring: copies of a quantised matrix, tangents, values next to zero,
gradients that need every bit of their planes."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import ops


def rnd(*shape, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return torch.randn(*shape, generator=g)


def through_torch(q, **to):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    with torch.serialization.safe_globals([ops.MXTensor]):
        return torch.load(f, weights_only=True, **to)


# ---------------------------------------------------------------- copies
@pytest.mark.parametrize("how", ["deepcopy", "torch.save", "host"])
def test_a_copy_outlives_the_original(how):
    x, w = rnd(20, 300, seed=1).cuda(), rnd(70, 300, seed=2).cuda()
    q = ops.mx_quantize(w)
    y, v = ops.mx_linear(x, q), q.dequantize()
    if how == "host":  # written on the host, read there, moved by hand
        h = through_torch(q, map_location="cpu")
        with pytest.raises(ValueError):
            ops.mx_linear(x, h)
        c = ops.MXTensor(h.buffer.cuda(), h.shape)
    else:
        c = copy.deepcopy(q) if how == "deepcopy" else through_torch(q)
    q.buffer.fill_(255)  # what stands there is nobody's matrix any more
    del q
    torch.cuda.synchronize()
    assert torch.equal(ops.mx_linear(x, c), y) and torch.equal(c.dequantize(), v)
    assert torch.equal(ops.mx_linear(ops.mx_quantize(x), c), y)


# ---------------------------------------------------------------- tangents
def test_duals_are_refused_and_their_primals_taken():
    import torch.autograd.forward_ad as fw
    t = rnd(40, 40).cuda()
    q = ops.mx_quantize(t)
    calls = (lambda x: ops.global_norm([t, x]), lambda x: ops.clip_by_global_norm([x], 1.0)[0][0],
             lambda x: ops.clip_by_global_norm([t], 1.0, use_norm=x[0, 0])[0][0],
             lambda x: ops.mx_quantize(x).dequantize(), lambda x: ops.mx_linear(x, q),
             lambda x: ops.mx_linear(t, q, bias=x[0]), lambda x: ops.mx_linear_grad(x, q, q)[0])
    for f in calls:
        want = f(t)
        with fw.dual_level():
            d = fw.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match="tangent"):
                f(d)
            assert torch.equal(f(d.detach()), want) and torch.equal(f(t), want)
