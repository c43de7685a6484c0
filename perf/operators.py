"""Cases that measure the tensor operators: the global gradient norm and the
clip by it, MXFP4 quantisation, the product of 4-bit operands and its
gradient.

run() computes a case in plain torch (own = False) or through
distributed_ddpg_amd.ops (own = True); exact() computes it in float64 from the
definitions.  Formats: OCP microscaling with E2M1 elements -- blocks of 32
along a row share a power-of-two scale 2^E, E = floor(log2(max |x|)) - 2, and
an element is one of 0 .5 1 1.5 2 3 4 6 (times 2^E), rounded to nearest with
ties to the even code, saturating at 6.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases
def net_shapes(S, A, h1, h2, critics):
    """One actor's and `critics` critics' parameter shapes (the checkpoint's
    tensors: their gradients are what a learner step clips)."""
    shapes = [(S, h1), (h1,), (h1, h2), (h2,), (h2, A)]
    for _ in range(critics):
        shapes += [(S, h1), (h1,), (A, h1), (h1,), (2 * h1, h2), (h2,), (h2, 1), (1,)]
    return shapes


def listed():
    return [
        # the default networks' gradients, every step of a small-batch learner: latency
        dict(name="norm_default", op="norm", S=4, A=1, h1=128, h2=200, critics=1, dtype="fp32"),
        # an ensemble of ten Humanoid-shaped critics kept in bf16
        dict(name="norm_ensemble", op="norm", S=376, A=17, h1=2048, h2=2048, critics=10,
             dtype="bf16"),
        # the synthetic benchmark's networks (S=64, A=16, 1024/1024), clipped before Adam
        dict(name="clip_bench", op="clip", S=64, A=16, h1=1024, h2=1024, critics=1, dtype="fp32",
             clip=1.0),
        # far wider networks with twin critics: bandwidth
        dict(name="clip_wide", op="clip", S=376, A=17, h1=8192, h2=8192, critics=2, dtype="bf16",
             clip=0.5),
        # one batch of Humanoid-shaped hidden activations
        dict(name="quantise_batch", op="quantise", rows=256, cols=376, dtype="fp16", turned=False),
        # a layer's weights in checkpoint order [in, out]: the blocks run down its columns
        dict(name="quantise_weights", op="quantise", rows=8192, cols=8192, dtype="fp32",
             turned=True),
        # action selection for one state: the weights' bytes and the launch
        dict(name="linear_act", op="linear", M=1, K=1024, N=1024, dtype="fp32", act="elu",
             bias=True),
        # a benchmark batch through the hidden layer
        dict(name="linear_bench", op="linear", M=4096, K=1024, N=1024, dtype="bf16", act="elu",
             bias=True),
        # no size a multiple of anything
        dict(name="linear_odd", op="linear", M=1000, K=777, N=1203, dtype="fp16", act="tanh",
             bias=True),
        # many environments through wide layers: the matrix pipe
        dict(name="linear_wide", op="linear", M=16384, K=8192, N=8192, dtype="bf16", act="none",
             bias=False),
        # a training step of the 400/300 network's hidden layer, ragged batch
        dict(name="train_small", op="train", M=1001, K=400, N=300, dtype="fp32", act="none",
             bias=True),
        # a training step of a wide layer
        dict(name="train_wide", op="train", M=8192, K=4096, N=4096, dtype="bf16", act="none",
             bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "quantise", "linear", "train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("norm", "clip"):
        case = dict(op=op, S=_log(rng, 1, 400), A=rng.randint(1, 20), h1=_log(rng, 7, 4096),
                    h2=_log(rng, 5, 4096), critics=_log(rng, 1, 10), dtype=dtype)
        if op == "clip":
            case["clip"] = rng.choice([0.01, 0.5, 1.0, 40.0])
        return case
    if op == "quantise":
        return dict(op=op, rows=_log(rng, 1, 8192), cols=_log(rng, 1, 8192), dtype=dtype,
                    turned=rng.random() < 0.4)
    if op == "linear":
        return dict(op=op, M=_log(rng, 1, 8192), K=_log(rng, 17, 8192), N=_log(rng, 1, 8192),
                    dtype=dtype, act=rng.choice(["none", "elu", "tanh"]), bias=rng.random() < 0.7)
    return dict(op=op, M=_log(rng, 1, 8192), K=_log(rng, 17, 4096), N=_log(rng, 5, 4096),
                dtype=dtype, act="none", bias=rng.random() < 0.7)


def work(case):
    e = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] in ("norm", "clip"):
        n = sum(math.prod(s) for s in net_shapes(case["S"], case["A"], case["h1"], case["h2"],
                                                 case["critics"]))
        if case["op"] == "norm":
            return {"bytes": n * e + 4, "flops": 2 * n}
        return {"bytes": 2 * n * e + 4, "flops": 3 * n}
    if case["op"] == "quantise":  # values in, the values they are held as out
        n = case["rows"] * case["cols"]
        return {"bytes": n * (e + 4), "flops": 3 * n}
    M, K, N = case["M"], case["K"], case["N"]
    q = 17 / 32  # bytes a 4-bit value takes, its share of the block's scale included
    b = 4 * N if case["bias"] else 0
    if case["op"] == "linear":
        return {"bytes": M * K * e + N * K * q + M * N * e + b, "flops": 2 * M * N * K}
    # x, w, dy in; y, dx, dw (fp32) and the bias gradient out
    return {"bytes": M * K * e + N * K * 4 + M * N * e + M * N * e + M * K * e + 4 * N * K + 2 * b,
            "flops": 6 * M * N * K}


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The case's tensors, the same for every form of it."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] in ("norm", "clip"):
        # gradients: each tensor of its own magnitude, weights' below the biases'
        out = []
        for s in net_shapes(case["S"], case["A"], case["h1"], case["h2"], case["critics"]):
            size = math.exp(float(torch.rand((), generator=g, device=dev)) * 3.0 - 6.0)
            t = torch.empty(s, dtype=dt, device=dev)
            t.copy_(randn(*s).mul_(size))
            out.append(t)
        return {"grads": out}
    if case["op"] == "quantise":
        R, C = case["rows"], case["cols"]
        if case["turned"]:  # weights in [in, out] order, seen as [out, in]
            w = (randn(C, R) / math.sqrt(C)).to(dt)
            return {"x": w.t()}
        x = randn(R, C)
        return {"x": torch.where(x < 0, torch.expm1(x), x).to(dt)}  # ELU outputs
    M, K, N = case["M"], case["K"], case["N"]
    x = randn(M, K)
    s = {"x": torch.where(x < 0, torch.expm1(x), x).to(dt),
         "w": (randn(K, N) / math.sqrt(K)).t(),  # fp32 master weights, checkpoint order [in, out]
         "bias": randn(N) * 0.1 if case["bias"] else None}
    if case["op"] == "train":
        s["dy"] = (randn(M, N) / M).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "linear":
        # an acting worker holds the published policy's weights quantised
        if own:
            from distributed_ddpg_amd import ops
            s["wq"] = ops.mx_quantize(s["w"])
        else:
            s["wv"] = _plain_mx(s["w"])
        del s["w"]
    return s


# ---------------------------------------------------------------- plain forms
def _plain_mx(x):
    """The values (fp32) that x's rows are held as in MXFP4."""
    R, K = x.shape
    pad = -K % 32
    v = torch.zeros(R, K + pad, dtype=torch.float32, device=x.device)
    v[:, :K] = x
    v = v.view(R, (K + pad) // 32, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    a = torch.ldexp(v, -e)
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)
    q = torch.ldexp(torch.where(a < 0, -m, m), e)
    q = torch.where(torch.isfinite(top), q, torch.full_like(q, float("nan")))
    return q.view(R, K + pad)[:, :K]


def _act(y, act):
    if act == "elu":
        return torch.where(y < 0, torch.exp(y) - 1, y)
    return torch.tanh(y) if act == "tanh" else y


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("norm", "clip"):
        n = torch.sqrt(sum((t.double() ** 2).sum() for t in s["grads"]))
        if op == "norm":
            return n.float()
        c = case["clip"]
        k = torch.where(n <= c, torch.ones_like(n), c / n)
        return [(t.float() * k.float()).to(t.dtype) for t in s["grads"]] + [n.float()]
    if op == "quantise":
        return _plain_mx(s["x"])
    dt = s["x"].dtype
    xv = _plain_mx(s["x"])
    wv = s["wv"] if op == "linear" else _plain_mx(s["w"])
    y = xv @ wv.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _act(y, case["act"]).to(dt)
    if op == "linear":
        return y
    dy = s["dy"].float()
    out = [y, (dy @ wv).to(dt), dy.t() @ xv]
    return out + [dy.sum(0)] if s["bias"] is not None else out


def run(s):
    if not own:
        return _plain(s)
    from distributed_ddpg_amd import ops
    case = s["case"]
    op = case["op"]
    if op == "norm":
        return ops.global_norm(s["grads"])
    if op == "clip":
        out, n = ops.clip_by_global_norm(s["grads"], case["clip"])
        return list(out) + [n]
    if op == "quantise":
        return ops.mx_dequantize(ops.mx_quantize(s["x"]))
    if op == "linear":
        return ops.mx_linear(s["x"], s["wq"], s["bias"], act=case["act"])
    # a training step: the weights moved since the last one, so both operands
    # are quantised, multiplied, and differentiated through (straight-through)
    wq, xq = ops.mx_quantize(s["w"]), ops.mx_quantize(s["x"])
    y = ops.mx_linear(xq, wq, s["bias"], act=case["act"], dtype=s["x"].dtype)
    dx, dw, db = ops.mx_linear_grad(s["dy"], xq, wq, bias=s["bias"] is not None)
    return [y, dx, dw] + ([db] if db is not None else [])


# ---------------------------------------------------------------- float64
def _exact_mx(x):
    """Element by element from the format's table: a value is the count of the
    rounding borders below it, a border going to the even code beside it."""
    R, K = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -K % 32)).reshape(R, -1, 32)
    top = v.abs().max(dim=2, keepdim=True).values
    # floor(log2): float64's exponent field (every positive float32 is normal there)
    e = (top.view(torch.int64) >> 52 & 2047) - 1023 - 2
    e = e.clamp(-127, 127)
    scale = ((e + 1023) << 52).view(torch.float64)
    a = (v / scale).abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False),
                       (3.5, True), (5.0, False)):
        code += ((a >= border) if up else (a > border)).long()
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    q = table[code] * torch.sign(v) * scale
    q = torch.where(torch.isfinite(top).expand_as(q), q, torch.full_like(q, math.nan))
    return q.reshape(R, -1)[:, :K]


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("norm", "clip"):
        n2 = torch.zeros((), dtype=torch.float64, device="cuda")
        for t in s["grads"]:
            n2 += torch.linalg.vector_norm(t.double()) ** 2
        n = float(n2) ** 0.5
        if op == "norm":
            return n2.sqrt()
        k = 1.0 if n <= case["clip"] else case["clip"] / n
        return [t.double() * k for t in s["grads"]] + [n2.sqrt()]
    if op == "quantise":
        return _exact_mx(s["x"])
    xv, wv = _exact_mx(s["x"]), _exact_mx(s["w"])
    y = torch.mm(xv, wv.t())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "elu":
        y = torch.where(y < 0, torch.expm1(y), y)
    elif case["act"] == "tanh":
        y = torch.tanh(y)
    if op == "linear":
        return y
    dy = s["dy"].double()
    out = [y, torch.mm(dy, wv), torch.mm(dy.t(), xv)]
    return out + [dy.sum(dim=0)] if s["bias"] is not None else out
