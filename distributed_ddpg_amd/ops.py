"""Tensor operators on torch tensors of the GPU: the global gradient norm and
the clip by it, MXFP4 quantisation, the product of quantised matrices and its
gradient (include/ddpg_hip.h, "tensor operators").

  global_norm(t_list)                         tf.global_norm
  clip_by_global_norm(t_list, clip_norm)      tf.clip_by_global_norm
  mx_quantize(x) -> MXTensor                  OCP MXFP4: blocks of 32 along a row
  mx_dequantize(q) -> tensor
  mx_linear(x, w, bias, act) -> tensor        act(x w^T + bias) in 4 bits
  mx_linear_grad(dy, x, w) -> dx, dw, db      straight-through gradient

Each call launches on torch's current stream of the tensors' device and
returns without waiting; results and workspaces come from torch's allocator, so
calls may be captured into a graph.  The operators have no autograd formula of
their own (the learner's gradients are explicit, as ActorNetwork.train's are): a
tensor that requires grad is refused while grad mode is on.  Arguments of the
wrong shape, type or device raise ValueError, the library's own refusals
DDPGError.
"""
import ctypes

import torch

from . import _lib
from ._lib import lib

_DTYPES = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "elu": _lib.ACT_ELU, "tanh": _lib.ACT_TANH}


def _check(rc):
    if rc < 0:
        raise _lib.DDPGError(rc, (lib.ddpg_global_error() or b"").decode(errors="replace"))


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _tensor(name, t):
    """t's dtype code, after the checks every operand shares."""
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s: expected a tensor, got %s" % (name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError("%s: expected a GPU tensor, got one on %s" % (name, t.device))
    code = _DTYPES.get(t.dtype)
    if code is None or t.layout is not torch.strided:
        raise ValueError("%s: %s is none of float32, bfloat16, float16" % (name, t.dtype))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad and the operator has no autograd formula; call it "
                         "under torch.no_grad() or pass .detach()" % name)
    return code


# ---------------------------------------------------------------- global norm
def _rows(t):
    """(cols, ld) of a tensor whose elements, in its own index order, are rows
    of adjacent elements a fixed distance apart; (0, 0) if it is dense in some
    index order (the operators do not care which); None if neither."""
    if t.is_contiguous():
        return 0, 0
    dims = [(st, n) for st, n in zip(t.stride(), t.shape) if n != 1]
    want = 1
    for st, n in sorted(dims):
        if st != want:
            break
        want *= n
    else:
        return 0, 0
    cols, i = 1, len(dims) - 1
    while i >= 0 and dims[i][0] == cols:
        cols *= dims[i][1]
        i -= 1
    if i < 0:
        return 0, 0
    ld, span = dims[i][0], dims[i][0]
    while i >= 0 and dims[i][0] == span:
        span *= dims[i][1]
        i -= 1
    return (cols, ld) if i < 0 else None


class _List:
    """The C form of a tensor list (None entries dropped)."""

    def __init__(self, name, tensors, inplace):
        self.kept = [t for t in tensors if t is not None]
        self.src, dt, cols, ld = [], [], [], []
        self.device = None
        strided = False
        for i, t in enumerate(self.kept):
            dt.append(_tensor("%s[%d]" % (name, i), t))
            if self.device is None:
                self.device = t.device
            elif t.device != self.device:
                raise ValueError("%s: tensors on %s and %s" % (name, self.device, t.device))
            if not t.is_contiguous():
                rc = _rows(t)
                if rc is None:
                    if inplace:
                        raise ValueError("%s[%d]: strides %s are neither dense nor evenly spaced "
                                         "rows" % (name, i, tuple(t.stride())))
                    t, rc = t.contiguous(), (0, 0)
                strided = strided or rc[0] > 0
                cols.append(rc[0])
                ld.append(rc[1])
            else:
                cols.append(0)
                ld.append(0)
            self.src.append(t)
        n = self.n = len(self.src)
        self.dtype = (ctypes.c_int * n)(*dt)
        self.ptr = (ctypes.c_void_p * n)(*[t.data_ptr() for t in self.src])
        self.count = (ctypes.c_int64 * n)(*[t.numel() for t in self.src])
        self.cols = (ctypes.c_int64 * n)(*cols) if strided else None
        self.ld = (ctypes.c_int64 * n)(*ld) if strided else None

    def need_device(self, name):
        if self.device is None:
            raise ValueError("%s: no tensor in the list" % name)
        return self.device

    def workspace(self):
        nb = lib.ddpg_global_norm_workspace(self.n)
        return torch.empty(nb, dtype=torch.uint8, device=self.device), nb


def global_norm(t_list):
    """sqrt of the sum of all elements' squares, a float32 scalar tensor.
    The sum runs in float64 in a fixed order.  Tensors may mix float32, bfloat16
    and float16 and be of any strides; None entries count nothing."""
    l = _List("t_list", t_list, False)
    dev = l.need_device("t_list")
    ws, nb = l.workspace()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    _check(lib.ddpg_global_norm(dev.index, _stream(dev), l.n, l.dtype, l.ptr, l.count, l.cols,
                                l.ld, ws.data_ptr(), nb, norm.data_ptr()))
    return norm


def clip_by_global_norm(t_list, clip_norm, use_norm=None, inplace=False):
    """(list_clipped, norm): each tensor times clip_norm / norm where norm =
    global_norm(t_list) exceeds clip_norm, unchanged (a copy) otherwise.

    use_norm: a float32 scalar tensor of the same device to use as the norm.
    inplace: write the results into t_list's own tensors (dense, or evenly
    spaced rows; no two may overlap).  None entries stay None.  A NaN norm
    makes every result NaN; an infinite one leaves zeros where the input is finite
    and NaN elsewhere."""
    t_list = list(t_list)
    clip_norm = float(clip_norm)
    if not clip_norm >= 0:
        raise ValueError("clip_norm %r is not a number >= 0" % clip_norm)
    l = _List("t_list", t_list, inplace)
    dev = l.need_device("t_list")
    if use_norm is not None:
        if _tensor("use_norm", use_norm) != _lib.FP32 or use_norm.numel() != 1 or (
                use_norm.device != dev):
            raise ValueError("use_norm: expected one float32 on %s" % dev)
        norm, ws, nb = use_norm, None, 0
    else:
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ws, nb = l.workspace()
    if inplace:
        out, dst = l.kept, l.ptr
    else:
        out = [torch.empty(t.shape, dtype=t.dtype, device=dev) if l.cols and l.cols[i]
               else torch.empty_like(t) for i, t in enumerate(l.src)]
        dst = (ctypes.c_void_p * l.n)(*[t.data_ptr() for t in out])
    _check(lib.ddpg_clip_by_global_norm(
        dev.index, _stream(dev), l.n, l.dtype, l.ptr, dst, l.count, l.cols, l.ld, clip_norm,
        None if use_norm is None else norm.data_ptr(), None if ws is None else ws.data_ptr(), nb,
        None if use_norm is not None else norm.data_ptr()))
    it = iter(out)
    return [None if t is None else next(it) for t in t_list], norm


# ---------------------------------------------------------------- MXFP4
class MXTensor:
    """A [rows, cols] matrix in MXFP4: 4-bit codes and a scale byte for 32 of
    them along a row, in the order the matrix instructions read (an opaque pair
    of byte buffers; .dequantize() gives the values).  17/32 byte a value."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes, scales, shape):
        self.codes, self.scales, self.shape = codes, scales, shape

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        return mx_dequantize(self, dtype)

    def __repr__(self):
        return "MXTensor(%d x %d, %s)" % (self.shape[0], self.shape[1], self.device)


def _matrix(name, t):
    code = _tensor(name, t)
    if t.dim() != 2:
        raise ValueError("%s: expected [rows, cols], got %s" % (name, tuple(t.shape)))
    return code


def _mx(name, q, cols=None, device=None):
    if not isinstance(q, MXTensor):
        raise ValueError("%s: expected an MXTensor (mx_quantize), got %s" % (name,
                                                                            type(q).__name__))
    if cols is not None and q.shape[1] != cols:
        raise ValueError("%s: expected [*, %d], got %s" % (name, cols, tuple(q.shape)))
    if device is not None and q.device != device:
        raise ValueError("%s is on %s, the other operand on %s" % (name, q.device, device))
    return q


def _mx_empty(rows, cols, device):
    tiles = -(-rows // 64) * -(-cols // 128)
    buf = torch.empty(tiles * 4352, dtype=torch.uint8, device=device)
    return MXTensor(buf[:tiles * 4096], buf[tiles * 4096:], (rows, cols))


def mx_quantize(x):
    """x [rows, cols] (float32, bfloat16 or float16, any strides) in MXFP4.

    Blocks of 32 values along a row share the scale 2^(floor(log2(max |x|)) - 2);
    each value becomes the nearest of 0 .5 1 1.5 2 3 4 6 times the scale, ties to
    the even code, larger ones 6.  A block that holds an infinity or a NaN is
    NaN as a whole."""
    code = _matrix("x", x)
    q = _mx_empty(x.shape[0], x.shape[1], x.device)
    _check(lib.ddpg_mx_quantize(x.device.index, _stream(x.device), code, x.data_ptr(), x.shape[0],
                                x.shape[1], x.stride(0), x.stride(1), q.codes.data_ptr(),
                                q.scales.data_ptr()))
    return q


def mx_dequantize(q, dtype=torch.float32):
    """The values q stands for, [rows, cols].  Exact in float32 and bfloat16;
    float16 rounds what lies outside its range."""
    _mx("q", q)
    if dtype not in _DTYPES:
        raise ValueError("dtype: %s is none of float32, bfloat16, float16" % dtype)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    _check(lib.ddpg_mx_dequantize(q.device.index, _stream(q.device), q.codes.data_ptr(),
                                  q.scales.data_ptr(), q.shape[0], q.shape[1], _DTYPES[dtype],
                                  out.data_ptr(), q.shape[1]))
    return out


def mx_linear(x, w, bias=None, act=None, dtype=None):
    """act(x w^T + bias), [M, N]: x [M, K] a tensor (quantised on the way) or an
    MXTensor, w [N, K] an MXTensor, bias [N], act None / "elu" / "tanh".  Sums in
    float32; the result is of x's type, or of dtype (float32 if x is an
    MXTensor)."""
    _mx("w", w)
    N, K = w.shape
    dev = w.device
    if act not in _ACTS:
        raise ValueError("act: %r is none of None, 'elu', 'tanh'" % (act,))
    if isinstance(x, MXTensor):
        xq, xp, xc, s0, s1 = _mx("x", x, K, dev), None, 0, 0, 0
        dtype = dtype or torch.float32
    else:
        xc = _matrix("x", x)
        if x.shape[1] != K:
            raise ValueError("x: expected [*, %d], got %s" % (K, tuple(x.shape)))
        if x.device != dev:
            raise ValueError("x is on %s, w on %s" % (x.device, dev))
        xq, xp, (s0, s1) = _mx_empty(x.shape[0], K, dev), x.data_ptr(), x.stride()
        dtype = dtype or x.dtype
    if dtype not in _DTYPES:
        raise ValueError("dtype: %s is none of float32, bfloat16, float16" % dtype)
    bc, bp = 0, None
    if bias is not None:
        bc = _tensor("bias", bias)
        if tuple(bias.shape) != (N,) or bias.device != dev:
            raise ValueError("bias: expected [%d] on %s, got %s on %s" % (
                N, dev, tuple(bias.shape), bias.device))
        bias = bias.contiguous()
        bp = bias.data_ptr()
    M = xq.shape[0]
    y = torch.empty((M, N), dtype=dtype, device=dev)
    _check(lib.ddpg_mx_linear(dev.index, _stream(dev), xc, xp, s0, s1, xq.codes.data_ptr(),
                              xq.scales.data_ptr(), M, K, w.codes.data_ptr(), w.scales.data_ptr(),
                              N, bc, bp, _ACTS[act], _DTYPES[dtype], y.data_ptr(), N))
    return y


def mx_linear_grad(dy, x, w, need=(True, True), bias=True):
    """(dx, dw, db) of mx_linear's product x w^T + bias (before act) for dy
    [M, N], with the values the MXTensors x [M, K] and w [N, K] stand for: dx = dy w
    of dy's type, dw = dy^T x and db = dy's column sums in float32.  The
    quantisation's own derivative is taken as 1 (straight-through), so dx and dw
    are the gradients of the matrices that were quantised.  need: whether dx,
    dw are wanted (None otherwise); bias: whether db is."""
    code = _matrix("dy", dy)
    dev = dy.device
    _mx("x", x, None, dev)
    _mx("w", w, x.shape[1], dev)
    (M, K), N = x.shape, w.shape[0]
    if tuple(dy.shape) != (M, N):
        raise ValueError("dy: expected [%d, %d], got %s" % (M, N, tuple(dy.shape)))
    need_dx, need_dw, bias = bool(need[0]), bool(need[1]), bool(bias)
    dx = torch.empty((M, K), dtype=dy.dtype, device=dev) if need_dx else None
    dw = torch.empty((N, K), dtype=torch.float32, device=dev) if need_dw else None
    db = torch.empty(N, dtype=torch.float32, device=dev) if bias else None
    nb = lib.ddpg_mx_linear_grad_workspace(code, M, N, K, need_dx, need_dw, bias)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _check(lib.ddpg_mx_linear_grad(
        dev.index, _stream(dev), code, dy.data_ptr(), dy.stride(0), dy.stride(1), M, N, K,
        x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
        dx.data_ptr() if need_dx else None, dw.data_ptr() if need_dw else None,
        db.data_ptr() if bias else None, ws.data_ptr(), nb))
    return dx, dw, db
