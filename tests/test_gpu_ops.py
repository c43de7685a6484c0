"""Tensor operators (distributed_ddpg_amd/ops.py) on the GPU against the
float64 oracle (oracle/ops_oracle.py).

Tolerances, from the arithmetic: a float32 sum of n products loses at most
2^-23 of the magnitudes' sum an addition (a matrix instruction may truncate), so
(n + 2) 2^-23 S; a rounding to type t half a step, finfo(t).eps / 2 of the value
(plus half the smallest subnormal); ELU 2^-22 and tanhf 2^-22 absolute.
Quantised values have to be equal."""
import math

import pytest
import torch

from oracle import ops_oracle as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from distributed_ddpg_amd import _lib, ops

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rnd(*shape, dt="fp32", seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(DT[dt])


def half_step(t, v):
    """A rounding of v to type t: half a step, also among the subnormals."""
    f = torch.finfo(t)
    return v.abs() * (f.eps / 2) * (1 + 2.0 ** -10) + f.smallest_normal * f.eps / 2 * (1 + 2.0 ** -10)


def close(got, want, tol):
    got = got.double().cpu()
    assert got.shape == want.shape
    both = torch.isnan(got) & torch.isnan(want)
    bad = ~both & ~((got - want).abs() <= tol) & ~(got == want)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


def same(got, want):
    got = got.double().cpu()
    ok = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert got.shape == want.shape and ok.all(), (got[~ok][:4], want[~ok][:4])


# ---------------------------------------------------------------- global norm
LISTS = {
    "one": [(1,)],
    "net": [(4, 128), (128,), (128, 200), (200,), (200, 1)],
    "ragged": [(7,), (3, 5), (0,), (16385,), (1,), (4095,), (33, 129), (2, 0, 3)],
    "many": [(1 + 37 * i % 501,) for i in range(230)],  # three tables
    "big": [(1 << 22,), (3,), (1025, 1023)],
}


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("name", sorted(LISTS))
def test_norm_and_clip(name, dt):
    kinds = ["fp32", "bf16", "fp16"] if dt == "mixed" else [dt]
    ts = [rnd(*s, dt=kinds[i % len(kinds)], seed=i) for i, s in enumerate(LISTS[name])]
    dev = [t.cuda() for t in ts]
    n = O.global_norm(ts)
    got = ops.global_norm(dev)
    assert got.shape == () and abs(float(got) - n) <= n * 2.0 ** -24 * (1 + 1e-6)
    for c in (n * 2 + 1, n * 0.3, 0.0, math.inf):
        want, _ = O.clip(ts, c)
        out, gn = ops.clip_by_global_norm(dev, c)
        assert torch.equal(gn, got)
        # clip_norm is a float32 at the C entry: 2^-24 of the scale
        for o, w, t in zip(out, want, ts):
            assert o.dtype == t.dtype
            close(o, w, half_step(t.dtype, w) + w.abs() * 2.0 ** -24)
        place = [t.clone() for t in dev]
        res, _ = ops.clip_by_global_norm(place, c, inplace=True)
        for r, p, o in zip(res, place, out):
            assert r is p and torch.equal(p, o)
        again, _ = ops.clip_by_global_norm(dev, c)
        assert all(torch.equal(a, o) for a, o in zip(again, out))


def test_norm_range_and_not_finite():
    for v in (1e30, 3e38, 1e-30, 1e-44):  # squares outside float32
        t = torch.full((1000,), v)
        n = O.global_norm([t])
        got = float(ops.global_norm([t.cuda()]))
        assert got == float(torch.tensor(n, dtype=torch.float64).float())
    x = rnd(100)
    for v in (math.inf, -math.inf, math.nan):
        t = x.clone()
        t[37] = v
        out, n = ops.clip_by_global_norm([t.cuda(), x.cuda()], 1.0)
        assert not math.isfinite(float(n)) and math.isnan(float(n)) == math.isnan(v)
        if math.isnan(v):
            assert all(o.isnan().all() for o in out)
        else:
            assert out[0][37].isnan() and int(out[0].isnan().sum()) == 1 and not out[1].any()


def test_norm_strides_none_and_use_norm():
    base = rnd(64, 96).cuda()
    views = [base[:, :40], base[:, 40:41], base[3:9, 50:60], base[:, 64:96].t(), None,
             base[::2, 41:49]]
    flat = [None if v is None else v.cpu().contiguous() for v in views]
    n = O.global_norm(flat)
    assert abs(float(ops.global_norm(views)) - n) <= n * 2.0 ** -23
    want, _ = O.clip(flat, 0.5)
    out, gn = ops.clip_by_global_norm(views, 0.5)
    for o, w in zip(out, want):
        if w is not None:
            close(o, w, half_step(torch.float32, w) * 2)
    # in place, rows of disjoint column ranges of one matrix
    work = base.clone()
    cols = [work[:, :40], work[:, 40:41], work[:, 41:90]]
    ops.clip_by_global_norm(cols, 0.5, inplace=True)
    ref, _ = O.clip([base[:, :90].cpu()], 0.5)
    close(work[:, :90], ref[0], half_step(torch.float32, ref[0]) * 2)
    assert torch.equal(work[:, 90:], base[:, 90:])  # the rest untouched
    three = base[:8, :8].reshape(2, 4, 8).permute(1, 0, 2)
    out, _ = ops.clip_by_global_norm([three], 1e9)
    assert torch.equal(out[0], three)
    exp = base[:1, :32].expand(5, 32)  # a broadcast input counts every copy
    assert abs(float(ops.global_norm([exp])) - O.global_norm([exp.cpu()])) <= 1e-6
    given = torch.tensor(8.0, device="cuda")
    out, gn = ops.clip_by_global_norm([base], 2.0, use_norm=given)
    assert gn is given
    close(out[0], base.double().cpu() / 4, half_step(torch.float32, base.double().cpu()))
    off = torch.arange(1001, dtype=torch.bfloat16, device="cuda")[1:]  # 2-byte aligned
    assert abs(float(ops.global_norm([off])) / O.global_norm([off.cpu()]) - 1) < 2.0 ** -23


def test_clip_in_place_is_seen_by_autograd():
    a = torch.ones(8, device="cuda", requires_grad=True)
    g = torch.full((8,), 3.0, device="cuda")
    y = a * g  # keeps g for its backward
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a], 1.0)
    ops.clip_by_global_norm([g], 1.0, inplace=True)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    with torch.no_grad():
        out, _ = ops.clip_by_global_norm([a], 1e9)
    assert torch.equal(out[0], a) and not out[0].requires_grad


def test_lists_refuse_what_has_no_dense_storage():
    a = torch.ones(4, 4, device="cuda")
    for bad in (a.to_sparse(), a.to_sparse_csr(), a.to("meta"), a.int(), a.cpu()):
        for ts in ([bad], [a, bad], [bad, a]):
            with pytest.raises(ValueError):
                ops.global_norm(ts)
            with pytest.raises(ValueError):
                ops.clip_by_global_norm(ts, 1.0)
    mixed = [2 * a, a.half(), a.bfloat16(), a.t()[1:], a.half()]  # 64 + 16 + 16 + 12 + 16 = 124
    assert abs(float(ops.global_norm(mixed)) - 124 ** 0.5) <= 12 * 2.0 ** -24


def test_negated_views_are_refused():
    """A float view whose memory holds the opposite sign."""
    z = torch.complex(torch.ones(64, 64), 2 * torch.ones(64, 64)).cuda().conj()
    wq = ops.mx_quantize(torch.ones(64, 64, device="cuda"))
    for v in (z.imag, z.imag[:1, :1]):
        assert v.is_neg()
        for f in (lambda: ops.clip_by_global_norm([v], 1.0), lambda: ops.global_norm([z.real, v]),
                  lambda: ops.mx_quantize(v), lambda: ops.mx_linear(v, wq),
                  lambda: ops.mx_linear_grad(v, wq, wq)):
            with pytest.raises(ValueError):
                f()
    same(ops.mx_quantize(z.imag.resolve_neg()).dequantize(), torch.full((64, 64), -2.0).double())
    same(ops.mx_quantize(z.real).dequantize(), torch.ones(64, 64).double())


def test_clip_refuses_overlap():
    b = torch.ones(64, 64, device="cuda")
    for bad in ([b, b], [b, b[0]], [b[:, :40], b[:, 39:]], [b.view(-1)[:100], b.view(-1)[99:]],
                [b[:1].expand(4, 64)]):
        with pytest.raises(_lib.DDPGError):
            ops.clip_by_global_norm(bad, 0.5, inplace=True)
    assert torch.equal(b, torch.ones_like(b))
    with pytest.raises(ValueError):  # neither dense nor even rows
        ops.clip_by_global_norm([b.view(4, 16, 64)[:, :3, :5]], 0.5, inplace=True)


# ---------------------------------------------------------------- quantise
def hard(rows, cols, dt, seed=0):
    """Values over many magnitudes, with borders, zeros and subnormals."""
    x = rnd(rows, cols, seed=seed)
    x *= torch.exp2(torch.randint(-10, 10, (rows, 1), generator=torch.Generator().manual_seed(1)).float())
    f = x.view(-1)
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 4.0, 0.0, -0.0, -0.75])
    f[::3] = grid[torch.arange(f[::3].numel()) % len(grid)]
    if rows > 4:
        x[1] = 0
        x[2] *= 1e-30
    return x.to(DT[dt])


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (16, 33), (17, 128), (64, 129),
                                       (65, 100), (130, 257), (1, 4097), (300, 64), (5, 2048)])
def test_quantise(rows, cols, dt):
    x = hard(rows, cols, dt)
    want = O.mx_values(x)
    q = ops.mx_quantize(x.cuda())
    assert q.shape == (rows, cols)
    same(q.dequantize(), want)
    for o in ("bf16", "fp16"):
        w = want.to(DT[o]).double()  # exact in bf16, one rounding in fp16
        same(q.dequantize(DT[o]), w)
    # down the columns of a matrix, with odd strides, unaligned
    same(ops.mx_quantize(x.t().contiguous().cuda().t()).dequantize(), want)
    wide = torch.zeros(rows, cols + 3, dtype=x.dtype, device="cuda")
    wide[:, 1:cols + 1] = x.cuda()
    same(ops.mx_quantize(wide[:, 1:cols + 1]).dequantize(), want)
    step = torch.zeros(rows * 2, cols * 3, dtype=x.dtype, device="cuda")
    step[::2, ::3] = x.cuda()
    same(ops.mx_quantize(step[::2, ::3]).dequantize(), want)
    same(ops.mx_quantize(x[:1].cuda().expand(rows, cols)).dequantize(), want[:1].expand(rows, cols))


def test_quantise_extremes():
    m = torch.finfo(torch.float32).max
    x = torch.zeros(8, 64)
    x[0, :32] = m
    x[0, 3] = -m / 7
    x[1, :4] = torch.tensor([2.0 ** -126, 2.0 ** -127, 2.0 ** -128, 2.0 ** -149])
    x[2, 0] = 2.0 ** -149
    x[3, 5], x[3, 40] = math.inf, 2.0
    x[4, 5], x[4, 40] = math.nan, 2.0
    x[5, 0], x[5, 1] = 1e30, 1e-30
    x[6] = -0.0
    x[7, 33] = -math.inf
    v = ops.mx_quantize(x.cuda()).dequantize().cpu()
    same(v, O.mx_values(x))
    assert v[3, :32].isnan().all() and v[3, 40] == 2 and v[4, :32].isnan().all()
    assert v[7, 32:].isnan().all() and not v[7, :32].any() and v[0].isfinite().all()


def test_empty():
    e = torch.empty(0, 40, device="cuda")
    assert ops.mx_quantize(e).dequantize().shape == (0, 40)
    w = ops.mx_quantize(rnd(5, 40).cuda())
    assert ops.mx_linear(e, w).shape == (0, 5)
    assert ops.mx_linear(rnd(3, 40).cuda(), ops.mx_quantize(e)).shape == (3, 0)
    z = ops.mx_quantize(torch.empty(5, 0, device="cuda"))
    b = rnd(5).cuda()
    y = ops.mx_linear(torch.empty(3, 0, device="cuda"), z, b)
    assert torch.equal(y, b.expand(3, 5))
    dx, dw, db = ops.mx_linear_grad(torch.empty(0, 5, device="cuda"), ops.mx_quantize(e), w)
    assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (5, 40)
    dx, dw, db = ops.mx_linear_grad(torch.empty(3, 0, device="cuda"),
                                    ops.mx_quantize(rnd(3, 40).cuda()), ops.mx_quantize(e))
    assert dx.shape == (3, 40) and not dx.any() and dw.shape == (0, 40) and db.shape == (0,)
    assert float(ops.global_norm([torch.empty(0, device="cuda")])) == 0
    out, n = ops.clip_by_global_norm([torch.empty(0, device="cuda")], 1.0)
    assert float(n) == 0 and out[0].shape == (0,)


# ---------------------------------------------------------------- product
def linear_tol(y, s, k, dt, extra=0.0):
    return s * (k + 2) * 2.0 ** -23 + 2.0 ** -22 * (1 + y.abs()) * extra + half_step(dt, y)


SHAPES = [(1, 32, 1), (1, 1, 1), (1, 128, 16), (1, 1024, 1024), (2, 130, 300), (5, 400, 17),
          (16, 256, 64), (17, 96, 65), (33, 511, 129), (64, 128, 128), (100, 777, 203),
          (128, 256, 256), (200, 2049, 255), (257, 384, 513), (300, 64, 1), (512, 1000, 1000)]


@pytest.mark.parametrize("dt,act,bias", [("fp32", "elu", "fp32"), ("bf16", None, None),
                                         ("fp16", "tanh", "bf16"), ("fp32", None, "fp16")])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(M, K, N, dt, act, bias):
    x, w = rnd(M, K, dt=dt, seed=1), rnd(N, K, seed=2, scale=K ** -0.5)
    b = None if bias is None else rnd(N, dt=bias, seed=3)
    xv, wv = O.mx_values(x), O.mx_values(w)
    want, s = O.linear(xv, wv, b, act)
    wq = ops.mx_quantize(w.cuda())
    bd = None if b is None else b.cuda()
    y = ops.mx_linear(x.cuda(), wq, bd, act)
    assert y.dtype == x.dtype
    close(y, want, linear_tol(want, s, K, x.dtype, 1.0 if act else 0.0))
    xq = ops.mx_quantize(x.cuda())
    assert torch.equal(ops.mx_linear(xq, wq, bd, act, dtype=x.dtype), y)
    turned = x.t().contiguous().cuda().t()  # strides of another order
    assert torch.equal(ops.mx_linear(turned, wq, bd, act), y)
    y32 = ops.mx_linear(xq, wq, bd, act)
    assert y32.dtype == torch.float32
    close(y32, want, linear_tol(want, s, K, torch.float32, 1.0 if act else 0.0))


def test_linear_nan_stays_in_its_row_and_column():
    M, K, N = 40, 200, 70
    x, w = rnd(M, K, seed=4), rnd(N, K, seed=5)
    x[7, 50], w[13, 150] = math.nan, math.inf
    y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda())).cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[7], want[:, 13] = True, True
    assert torch.equal(y.isnan(), want)


def test_linear_large_and_tiny_scales():
    x, w = rnd(20, 96, seed=6) * 1e30, rnd(24, 96, seed=7) * 1e-36
    xv, wv = O.mx_values(x), O.mx_values(w)
    want, s = O.linear(xv, wv)
    close(ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda())), want,
          linear_tol(want, s, 96, torch.float32))


# ---------------------------------------------------------------- gradient
@pytest.mark.parametrize("M", [1, 100, 2048])  # each kernel's epilogue
def test_activations_over_their_range(M):
    """act(0 + bias): the activation alone.  elu: exp(x) - 1, its argument's rounding
    moves it by |x| e^x 2^-24 <= 2^-25, exp by 2^-23, the difference by 2^-25.  tanh by
    1 - 2 r: e's error enters as 2 (r - r^2) (2^-23 + 2 |x| 2^-24) <= 2^-23, the sum's and
    r's as 2 r (2^-24 + 2^-23) <= 0.81 2^-23 (r < 0.27), the last rounding as 2^-25; its
    polynomial, below 0.5, is within 2^-23 of the value (and half a step)."""
    b = torch.cat([torch.linspace(-12, 12, 1999), torch.linspace(-0.6, 0.6, 2001),
                   torch.logspace(-38, 2, 47), -torch.logspace(-38, 2, 47),
                   torch.tensor([0.0, -0.0, 0.5, -0.5, 88.0, -104.0, 1e30, -1e30, math.inf,
                                 -math.inf, math.nan])]).float()
    x, wq = torch.zeros(M, 1, device="cuda"), ops.mx_quantize(torch.zeros(len(b), 1, device="cuda"))
    t = b.double()
    for act, want, tol in (("elu", torch.where(t < 0, torch.expm1(t), t),
                            torch.where(t < 0, 2.0 ** -22, 0.0)),
                           ("tanh", torch.tanh(t), torch.where(t.abs() < 0.5,
                                                               t.abs() * 1.5 * 2.0 ** -23,
                                                               2.25 * 2.0 ** -23))):
        y = ops.mx_linear(x, wq, b.cuda(), act).cpu().double()
        assert torch.equal(y[0], y[-1]) or torch.equal(y[0].isnan(), y[-1].isnan())
        for r in (y[0], y[-1]):
            assert torch.equal(r.isnan(), t.isnan())
            err = (r - want).abs()[:-1]
            err = torch.where(want[:-1] == r[:-1], 0.0, err)  # the infinite ones
            assert (err <= tol[:-1] + 2.0 ** -126).all(), (act, float((err - tol[:-1]).max()))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 300, 200), (3, 64, 64), (64, 32, 128),
                                   (65, 129, 63), (100, 400, 300), (1001, 400, 300),
                                   (256, 256, 256), (513, 257, 1025)])
def test_linear_grad(M, K, N, dt):
    x, w, dy = rnd(M, K, seed=1), rnd(N, K, seed=2), rnd(M, N, dt=dt, seed=3)
    xv, wv = O.mx_values(x), O.mx_values(w)
    want, s = O.linear_grad(dy, xv, wv)
    xq, wq = ops.mx_quantize(x.cuda()), ops.mx_quantize(w.cuda())
    got = ops.mx_linear_grad(dy.cuda(), xq, wq)
    n = (N, M, M)
    types = (dy.dtype, torch.float32, torch.float32)
    for g, v, a, k, t in zip(got, want, s, n, types):
        assert g.dtype == t
        close(g, v, a * (3 * k + 2) * 2.0 ** -23 + half_step(t, v))
    turned = ops.mx_linear_grad(dy.t().contiguous().cuda().t(), xq, wq)
    assert all(torch.equal(a, b) for a, b in zip(turned, got))
    dx, dw, db = ops.mx_linear_grad(dy.cuda(), xq, wq, need=(True, False), bias=False)
    assert torch.equal(dx, got[0]) and dw is None and db is None
    dx, dw, db = ops.mx_linear_grad(dy.cuda(), xq, wq, need=(False, True), bias=False)
    assert torch.equal(dw, got[1]) and dx is None and db is None
    dx, dw, db = ops.mx_linear_grad(dy.cuda(), xq, wq, need=(False, False))
    assert torch.equal(db, got[2]) and dx is None and dw is None


def test_linear_grad_by_differences():
    """The product is linear in x's and w's values: along a direction that keeps
    every value on the grid, (L(x + h u) - L(x)) / h is the gradient's share."""
    M, K, N = 9, 64, 12
    g = torch.Generator().manual_seed(0)
    grid = torch.tensor([-4.0, -2.0, -1.0, 0.0, 1.0, 2.0, 4.0])
    x = grid[torch.randint(0, 7, (M, K), generator=g)]
    w = grid[torch.randint(0, 7, (N, K), generator=g)]
    x[:, ::32] = 4.0  # every block's scale is 1
    w[:, ::32] = 4.0
    dy = grid[torch.randint(0, 7, (M, N), generator=g)]
    xq, wq = ops.mx_quantize(x.cuda()), ops.mx_quantize(w.cuda())
    dx, dw, _ = ops.mx_linear_grad(dy.cuda(), xq, wq)

    def loss(x, w):
        y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()))
        return float((y.double().cpu() * dy.double()).sum())

    for i, j in ((0, 1), (4, 33), (8, 63)):
        for base, other in ((-1.0, 1.0), (2.0, 3.0)):
            a, b = x.clone(), x.clone()
            a[i, j], b[i, j] = base, other
            assert (loss(b, w) - loss(a, w)) / (other - base) == float(dx[i, j])
            a, b = w.clone(), w.clone()
            a[i, j], b[i, j] = base, other
            assert (loss(x, b) - loss(x, a)) / (other - base) == float(dw[i, j])


def test_linear_grad_not_finite():
    M, K, N = 20, 40, 30
    x, w, dy = rnd(M, K, seed=1).abs() + 1, rnd(N, K, seed=2).abs() + 1, rnd(M, N, seed=3)
    dy[3, 4], dy[5, 6] = math.inf, math.nan
    dy[7, 8] = torch.finfo(torch.float32).max
    xq, wq = ops.mx_quantize(x.cuda()), ops.mx_quantize(w.cuda())
    dx, dw, db = (t.cpu() for t in ops.mx_linear_grad(dy.cuda(), xq, wq))
    assert (dx[3] == math.inf).all() and dx[5].isnan().all() and dx[:3].isfinite().all()
    assert (dw[4] == math.inf).all() and dw[6].isnan().all()
    assert db[4] == math.inf and db[6].isnan() and db[8] == dy[:, 8].double().sum().float()


# ---------------------------------------------------------------- together
def train_step(x, w, b, dy, clip):
    xq, wq = ops.mx_quantize(x), ops.mx_quantize(w)
    y = ops.mx_linear(xq, wq, b, "elu", dtype=x.dtype)
    dx, dw, db = ops.mx_linear_grad(dy, xq, wq)
    (dw, db), n = ops.clip_by_global_norm([dw, db], clip, inplace=True)
    return y, dx, dw, db, n


@pytest.mark.parametrize("M,K,N", [(1, 128, 200), (257, 400, 300)])
def test_a_step_streamed_and_captured(M, K, N):
    """The operators as a training step uses them: eagerly, on another stream,
    and replayed from two graphs with eager work between the replays."""
    x, w, b, dy = (t.cuda() for t in (rnd(M, K, dt="bf16"), rnd(K, N).t(), rnd(N),
                                      rnd(M, N, dt="bf16")))
    want = [t.clone() for t in train_step(x, w, b, dy, 0.1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train_step(x, w, b, dy, 0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = train_step(x, w, b, dy, 0.1)
        graphs.append((g, out))
    x0 = x.clone()
    for i in range(4):
        x.copy_(x0 * (i + 1))
        want = [t.clone() for t in train_step(x, w, b, dy, 0.1)]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want, out))


def test_two_streams_at_once():
    ts = [rnd(1 << 20, seed=i).cuda() for i in range(4)]
    w = ops.mx_quantize(rnd(512, 512).cuda())
    xs = [rnd(300, 512, seed=i).cuda() for i in range(4)]
    want = [(ops.global_norm([t]).clone(), ops.mx_linear(x, w).clone()) for t, x in zip(ts, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(3):
        for st, t, x in zip(streams, ts, xs):
            with torch.cuda.stream(st):
                got.append((ops.global_norm([t]), ops.mx_linear(x, w)))
    torch.cuda.synchronize()
    for i, (n, y) in enumerate(got):
        assert torch.equal(n, want[i % 4][0]) and torch.equal(y, want[i % 4][1])


# ---------------------------------------------------------------- large
def dev64(t):
    return t.double().cuda()


@pytest.mark.parametrize("dt,act", [("fp32", "elu"), ("bf16", None), ("fp16", "tanh")])
@pytest.mark.parametrize("M,K,N", [(1025, 300, 1100),   # 64 x 64 tiles
                                   (2001, 300, 1703),   # 128 x 128
                                   (2500, 2049, 1600),
                                   (4001, 200, 4099),   # 256 x 256
                                   (4096, 1100, 4352)])
def test_linear_tiles(M, K, N, dt, act):
    x, w, b = rnd(M, K, dt=dt, seed=1), rnd(N, K, seed=2, scale=K ** -0.5), rnd(N, seed=3)
    xv, wv = dev64(O.mx_values(x)), dev64(O.mx_values(w))
    want = O.act(xv @ wv.T + dev64(b), act)
    s = xv.abs() @ wv.abs().T + dev64(b).abs()
    y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()), b.cuda(), act)
    assert y.dtype == DT[dt]
    err = (y.double() - want).abs()
    assert (err <= linear_tol(want, s, K, DT[dt], 1.0 if act else 0.0)).all(), float(err.max())


@pytest.mark.parametrize("M,K,N,dt", [(700, 650, 900, "fp16"),     # 64 x 64 tiles
                                      (1100, 900, 1050, "fp16"),   # 128 x 128
                                      (2050, 2049, 2047, "bf16"),
                                      (8192, 4096, 64, "bf16"),    # and dW in 11 splits
                                      (8190, 65, 4095, "fp32"),
                                      (4099, 2051, 2040, "fp32"),  # 256 x 256, dW in 2 splits
                                      (16001, 300, 4096, "fp32"),  # in 4
                                      (8000, 17, 5, "fp32")])      # 32 x 32, dW in 12 splits
def test_linear_grad_tiles(M, K, N, dt):
    x, w, dy = rnd(M, K, seed=1), rnd(N, K, seed=2), rnd(M, N, dt=dt, seed=3)
    xv, wv, d = dev64(O.mx_values(x)), dev64(O.mx_values(w)), dev64(dy)
    want = (d @ wv, d.T @ xv, d.sum(0))
    s = (d.abs() @ wv.abs(), d.abs().T @ xv.abs(), d.abs().sum(0))
    xq, wq, dyd = ops.mx_quantize(x.cuda()), ops.mx_quantize(w.cuda()), dy.cuda()
    got = ops.mx_linear_grad(dyd, xq, wq)
    for g, v, a, k, t in zip(got, want, s, (N, M, M), (dy.dtype, torch.float32, torch.float32)):
        err = (g.double() - v).abs()
        assert (err <= a * (3 * k + 2) * 2.0 ** -23 + half_step(t, v)).all(), float(err.max())
    for _ in range(3):  # whichever split comes last
        assert all(torch.equal(a, b) for a, b in zip(ops.mx_linear_grad(dyd, xq, wq), got))
    dx, _, _ = ops.mx_linear_grad(dyd, xq, wq, need=(True, False), bias=False)
    _, dw, _ = ops.mx_linear_grad(dyd, xq, wq, need=(False, True), bias=False)
    assert torch.equal(dx, got[0]) and torch.equal(dw, got[1])


def test_offsets_past_32_bits():
    big = torch.empty((1 << 32) + 4096, dtype=torch.bfloat16, device="cuda")
    x = rnd(17, 200, dt="bf16", seed=8)
    far = big.as_strided((17, 200), (1 << 28, 1))
    far.copy_(x.cuda())
    same(ops.mx_quantize(far).dequantize(), O.mx_values(x))
    wq = ops.mx_quantize(rnd(40, 200).cuda())
    assert torch.equal(ops.mx_linear(far, wq), ops.mx_linear(x.cuda(), wq))
    turned = big.as_strided((200, 17), (1, 1 << 28))
    same(ops.mx_quantize(turned).dequantize(), O.mx_values(x.t()))
    assert float(ops.global_norm([far])) == float(ops.global_norm([x.cuda()]))
    dy = big.as_strided((17, 40), (1 << 28, 1))
    dy.copy_(x[:, :40].cuda())
    xq = ops.mx_quantize(x.cuda())
    a = ops.mx_linear_grad(dy, xq, wq)
    b = ops.mx_linear_grad(x[:, :40].cuda(), xq, wq)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    big.zero_()
    big[0], big[1 << 31], big[-1] = 2.0, 3.0, 6.0
    assert float(ops.global_norm([big])) == 7.0
    ops.clip_by_global_norm([big], 3.5, inplace=True)
    assert [float(big[i]) for i in (0, 1 << 31, -1)] == [1.0, 1.5, 3.0]
