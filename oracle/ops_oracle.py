"""Float64 restatement of the tensor operators (include/ddpg_hip.h, "tensor
operators") on CPU tensors: global norm, clip, MXFP4 values, the product of
quantised matrices and its straight-through gradient.  Written from the
definitions, element by element."""
import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def global_norm(ts):
    return sum(float((t.double() ** 2).sum()) for t in ts if t is not None) ** 0.5


def clip(ts, c, norm=None):
    n = global_norm(ts) if norm is None else norm
    s = 1.0 if n <= c else (c / n if n == n else float("nan"))
    return [None if t is None else t.double() * s for t in ts], n


def mx_values(x):
    """The values (float64) that the rows of x are held as in MXFP4."""
    rows, cols = x.shape
    xd = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64)
    xd[:, :cols] = x.double().cpu()
    b = xd.reshape(rows, -1, 32)
    top = b.abs().amax(dim=-1, keepdim=True) if b.numel() else b[..., :1]
    finite = torch.isfinite(top)
    # floor(log2(top)) by comparison with powers of two
    e = torch.floor(torch.log2(torch.where(finite & (top > 0), top, torch.ones_like(top))))
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(top > 0, e - 2, torch.full_like(e, -127.0)).clamp(-127, 127)
    a = (b / torch.exp2(e)).abs()
    best = torch.zeros_like(a)
    gap = torch.full_like(a, float("inf"))
    for code, v in enumerate(E2M1):
        d = (a - v).abs()
        # nearer, or as near with an even code
        take = (d < gap) | ((d == gap) & (code % 2 == 0))
        best = torch.where(take, torch.full_like(best, v), best)
        gap = torch.minimum(gap, d)
    q = torch.copysign(best, b) * torch.exp2(e)
    q = torch.where(finite, q, torch.full_like(q, float("nan")))
    return q.reshape(rows, -1)[:, :cols]


def act(y, name):
    if name == "elu":
        return torch.where(y < 0, torch.expm1(y), y)
    return torch.tanh(y) if name == "tanh" else y


def linear(xv, wv, bias=None, name=None):
    """(result, sum of the products' magnitudes) for values xv [M,K], wv [N,K]."""
    y, s = xv @ wv.T, xv.abs() @ wv.abs().T
    if bias is not None:
        y, s = y + bias.double().cpu(), s + bias.double().cpu().abs()
    return act(y, name), s


def linear_grad(dy, xv, wv):
    """((dx, dw, db), (their sums of magnitudes))."""
    d = dy.double().cpu()
    return ((d @ wv, d.T @ xv, d.sum(0)),
            (d.abs() @ wv.abs(), d.abs().T @ xv.abs(), d.abs().sum(0)))
