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


# ---------------------------------------------------------------- activations
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 100, 2048, 4096, 8192])  # rows; tiles of 32, 64, 128, 256
def test_activations_next_to_zero(M, dt):
    """act(0 + bias) relative to its value.  ELU: x + x^2 p(x) above -0.5, p within
    2^-26 / 0.64 and five roundings of terms at most 0.27 of the value, one of the whole:
    2^-23; below, |y| >= 0.39: the exponential's 2^-24, its argument's |x| e^x
    (2^-24 + 2^-26) and the difference's 2^-25 are under 2^-23 absolute, 2.8 2^-23 of the value.
    tanh below 0.5 as ELU: 1.5 2^-23; above, where it is at least 0.46, 2.25 2^-23 absolute:
    5 2^-23 of the value.  Then one rounding to dt.

    ELU for 16 bits: the smaller of e^x - 1 + 2^-23, off by at most 1.5 2^-23, and x + x^2 / 2,
    at most x^2 / 6 (1 + |x|) of the value above it.  The second is the smaller up to
    |x|^3 / 6 <= 1.5 2^-23, |x| <= 0.0103: 2^-15.7 of the value (roundings 2^-23 of it); behind that the
    first's 1.5 2^-23 is less of it still."""
    n = 700 if M < 8192 else 8300
    small = torch.logspace(-37, -0.302, n // 2, dtype=torch.float64).float()
    x = torch.cat([-small, small, -torch.linspace(0.4, 0.6, 201), torch.tensor([-0.0, 0.0])])
    t = x.double()
    zero = torch.zeros(M, 1, device="cuda")
    wq = ops.mx_quantize(torch.zeros(len(x), 1, device="cuda"))
    f = torch.finfo(dt)
    for act, want, rel in (
            ("elu", torch.where(t < 0, torch.expm1(t), t),
             (torch.where(t > -0.5, 1.0, 2.8) * 2.0 ** -23 if dt is torch.float32
              else 2.0 ** -15.6) * (t < 0)),
            ("tanh", torch.tanh(t), torch.where(t.abs() < 0.5, 1.5 * 2.0 ** -23, 5 * 2.0 ** -23))):
        y = ops.mx_linear(zero, wq, x.cuda(), act, dtype=dt)
        assert (y == y[0]).all()  # every row, whichever part of a tile it is in
        err = (y[0].cpu().double() - want).abs()
        half = 0 if dt is torch.float32 else f.eps / 2 * (1 + 2.0 ** -12)
        tol = want.abs() * (rel + half) + f.smallest_normal * f.eps
        assert (err <= tol).all(), (act, x[err > tol][:5], y[0].cpu()[err > tol][:5])
    # and not finite: the same in every row
    odd = torch.tensor([float("nan"), float("inf"), -float("inf")] * 3).cuda()
    wq = ops.mx_quantize(torch.zeros(9, 1, device="cuda"))
    y = ops.mx_linear(zero, wq, odd, "elu", dtype=dt).cpu()
    assert y[:, ::3].isnan().all() and (y[:, 1::3] == float("inf")).all() and (y[:, 2::3] == -1).all()
    y = ops.mx_linear(zero, wq, odd, "tanh", dtype=dt).cpu()
    assert y[:, ::3].isnan().all() and (y[:, 1::3] == 1).all() and (y[:, 2::3] == -1).all()


# ---------------------------------------------------------------- gradient
def integers(rows, cols, seed):
    """Values that MXFP4 holds exactly under a scale of 1."""
    g = torch.Generator().manual_seed(seed)
    t = torch.tensor([-4.0, -2.0, -1.0, 1.0, 2.0, 3.0, 4.0, 6.0])[
        torch.randint(0, 8, (rows, cols), generator=g)]
    t[:, ::32] = 6.0
    return t.cuda()


# (M, K, N): tile, splits of dX and dW with three planes
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,K,N", [(1001, 400, 300),    # 32, 1 and 2
                                   (513, 257, 1025),    # 32, 2 and 1
                                   (700, 650, 900),     # 64, 2 and 2
                                   (30000, 100, 60),    # 64, 1 and 32
                                   (1100, 900, 1050),   # 128, 2 and 2
                                   (2000, 1100, 1300),  # 128, 1 and 1
                                   (8190, 65, 4095),    # 128, 2 and 4
                                   (20000, 200, 200),   # 128, 1 and 32
                                   (2050, 2049, 2047),  # 256, 2 and 2
                                   (4099, 2051, 2040)])  # 256, 1 and 2
def test_every_plane_of_dy_counts(M, K, N, dt):
    """dY with at most four values a row (dX) or a column (dW), each 2^j (1 + 2^-9 + 2^-18)
    (fp16: without the last) -- a bit in every plane -- against integers up to 6: a
    sum has at most 5 bits above and 18 below the point, so float32 holds all of its
    partial sums and the results are exact.  A lost plane, or one that meets
    another depth step's operand, shows."""
    x, w = integers(M, K, 1), integers(N, K, 2)
    xq, wq = ops.mx_quantize(x), ops.mx_quantize(w)
    assert torch.equal(xq.dequantize(), x) and torch.equal(wq.dequantize(), w)
    v = 1 + 2.0 ** -9 + (2.0 ** -18 if dt is torch.float32 else 0)
    g = torch.Generator().manual_seed(3)
    dy = torch.zeros(M, N)
    for _ in range(4):  # a power of two a row
        dy[torch.arange(M), torch.randint(0, N, (M,), generator=g)] = v
    dy = (dy * torch.exp2((torch.arange(M) % 5).float())[:, None]).cuda().to(dt)
    dx, _, db = ops.mx_linear_grad(dy, xq, wq)
    assert torch.equal(dx, (dy.double() @ w.double()).to(dt))
    dy = torch.zeros(N, M)
    for _ in range(4):
        dy[torch.arange(N), torch.randint(0, M, (N,), generator=g)] = v
    dy = (dy * torch.exp2(-(torch.arange(N) % 5).float())[:, None]).t().cuda().to(dt)
    _, dw, db = ops.mx_linear_grad(dy, xq, wq)
    assert torch.equal(dw, (dy.double().t() @ x.double()).float())
    assert torch.equal(db, dy.double().sum(0).float())


@pytest.mark.parametrize("e", [-60, -100, -110, -115, -120, -126, -130, -140])
def test_a_tiny_gradient(e):
    """float32 dY next to bfloat16's smallest number 2^-133: whole down to 2^-110, below
    it rounded to a multiple of 2^-133.  The sums are float32's, subnormal ones too."""
    M, K, N = 9, 70, 33
    x, w = integers(M, K, 1), integers(N, K, 2)
    dy = (rnd(M, N, seed=5).double() * 2.0 ** e).float().cuda()
    dx, dw, db = ops.mx_linear_grad(dy, ops.mx_quantize(x), ops.mx_quantize(w))
    d = dy.double()
    for got, want, s, k, m in ((dx, d @ w.double(), d.abs() @ w.double().abs(), N, 6),
                               (dw, d.t() @ x.double(), d.abs().t() @ x.double().abs(), M, 6),
                               (db, d.sum(0), d.abs().sum(0), M, 0)):
        tol = s * (3 * k + 2) * 2.0 ** -23 + k * m * 2.0 ** -134 + (3 * k + 2) * 2.0 ** -149
        assert ((got.double() - want).abs() <= tol).all()


# ---------------------------------------------------------------- clip
def test_a_norm_outside_float32():
    """The norm of float32 values can overflow float32, never float64: the clip scales by
    it all the same.  A norm given as float32 infinity leaves zeros."""
    x = torch.full((1000,), 3e38).cuda()
    n = float(x[0].double()) * 1000 ** 0.5
    out, norm = ops.clip_by_global_norm([x], 1e38)
    assert torch.isinf(norm)
    c = float(torch.tensor(1e38, dtype=torch.float32).double())
    want = float(x[0].double()) * (c / n)
    assert ((out[0].double() - want).abs() <= want * (2.0 ** -24 + 2.0 ** -50)).all()
    out, _ = ops.clip_by_global_norm([x], 1e38, use_norm=norm)
    assert not out[0].any()
    x[7] = float("inf")
    out, norm = ops.clip_by_global_norm([x], float("inf"))  # the norm alone
    assert torch.isinf(norm) and torch.equal(out[0], x)
    out, norm = ops.clip_by_global_norm([x], 1.0)
    assert out[0][7].isnan() and not out[0][:7].any() and not out[0][8:].any()
    x[7] = float("nan")
    out, norm = ops.clip_by_global_norm([x], float("inf"))
    assert norm.isnan() and out[0].isnan().all()
