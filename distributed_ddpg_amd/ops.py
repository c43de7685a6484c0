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
tensor that requires grad is refused while grad mode is on, one with a
forward-mode tangent always.  Arguments of the wrong shape, type or device raise
ValueError, the library's own refusals DDPGError.
"""
import operator
from array import array

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import lib

_DTYPES = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "elu": _lib.ACT_ELU, "tanh": _lib.ACT_TANH}


def _check(rc):
    if rc < 0:
        raise _lib.DDPGError(rc, (lib.ddpg_global_error() or b"").decode(errors="replace"))


# the raw handle of torch's current stream on a device ordinal
_stream = torch._C._cuda_getCurrentRawStream


def _has_tangent(t):
    return forward_ad.unpack_dual(t).tangent is not None


def _tensor(name, t):
    """t's dtype code, after the checks every operand shares."""
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s: expected a tensor, got %s" % (name, type(t).__name__))
    if forward_ad._current_level >= 0 and _has_tangent(t):
        raise ValueError("%s carries a forward-mode tangent and the operator has no formula for "
                         "it; pass .detach()" % name)
    if not t.is_cuda:
        raise ValueError("%s: expected a GPU tensor, got one on %s" % (name, t.device))
    code = _DTYPES.get(t.dtype)
    if code is None or t.layout is not torch.strided:
        raise ValueError("%s: %s is none of float32, bfloat16, float16" % (name, t.dtype))
    if t.is_neg():
        raise ValueError("%s is a negated view (of a conjugate's imaginary part); pass "
                         ".resolve_neg()" % name)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad and the operator has no autograd formula; call it "
                         "under torch.no_grad() or pass .detach()" % name)
    return code


# ---------------------------------------------------------------- global norm
def _rows(t):
    """(cols, ld) of a tensor whose elements, in its own index order, are rows
    of adjacent elements a fixed distance apart; (0, 0) if it is dense in some
    index order (the operators do not care which); None if neither, or for rows
    longer than a kernel counts."""
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
    return (cols, ld) if i < 0 and cols < 1 << 31 else None


class _List:
    """The C form of a tensor list (None entries dropped)."""

    def __init__(self, tensors, inplace):
        self.src = src = [t for t in tensors if t is not None]
        if not src:
            raise ValueError("t_list: no tensor in the list")
        # whole-list checks (a list has hundreds of tensors); what fails one is
        # named by the tensor's own check (a sparse one has no data_ptr)
        try:
            dt = {t.dtype for t in src}
            dt = (array("i", [_DTYPES[dt.pop()]]) * len(src) if len(dt) == 1
                  else array("i", [_DTYPES[t.dtype] for t in src]))
            index = {t.get_device() for t in src}
            self.ptr = array("Q", [t.data_ptr() for t in src])
            fine = len(index) == 1 and min(index) >= 0 and not (
                any([t.requires_grad or t.is_neg() for t in src]) if torch.is_grad_enabled()
                else any(map(torch.Tensor.is_neg, src))) and not (
                forward_ad._current_level >= 0 and any(map(_has_tangent, src)))
        except (AttributeError, KeyError, TypeError, RuntimeError):
            fine = False
        if not fine:
            for i, t in enumerate(src):
                _tensor("t_list[%d]" % i, t)
            raise ValueError("t_list: tensors on %s" % " and ".join(
                sorted({str(t.device) for t in src})))
        self.index = index.pop()
        self.kept = src
        cols = ld = None
        if not all([t.is_contiguous() for t in src]):
            self.src = src = list(src)
            cols, ld = array("q", bytes(8 * len(src))), array("q", bytes(8 * len(src)))
            for i, t in enumerate(src):
                rc = _rows(t)
                if rc is None and inplace:
                    raise ValueError("t_list[%d]: strides %s are neither dense nor evenly spaced "
                                     "rows" % (i, tuple(t.stride())))
                if rc is None:
                    src[i] = t.contiguous()
                    self.ptr[i] = src[i].data_ptr()
                else:
                    cols[i], ld[i] = rc
        self.cols = cols
        self._held = (dt, cols, ld, array("q", [t.numel() for t in src]))
        self.n = len(src)
        addr = lambda a: None if a is None else a.buffer_info()[0]
        self.dtype, cols, ld, self.count = [addr(a) for a in self._held]
        self.rows = (cols, ld)
        self.ws_bytes = lib.ddpg_global_norm_workspace(self.n)

    def empty(self, n, dtype):
        return self.kept[0].new_empty(n, dtype=dtype)


def global_norm(t_list):
    """sqrt of the sum of all elements' squares, a float32 scalar tensor.
    The sum runs in float64 in a fixed order.  Tensors may mix float32, bfloat16
    and float16 and be of any strides; None entries count nothing."""
    l = _List(t_list, False)
    norm, ws = l.empty((), torch.float32), l.empty(l.ws_bytes, torch.uint8)
    _check(lib.ddpg_global_norm(l.index, _stream(l.index), l.n, l.dtype, l.ptr.buffer_info()[0],
                                l.count, *l.rows, ws.data_ptr(), l.ws_bytes, norm.data_ptr()))
    return norm


def clip_by_global_norm(t_list, clip_norm, use_norm=None, inplace=False):
    """(list_clipped, norm): each tensor times clip_norm / norm where norm =
    global_norm(t_list) exceeds clip_norm (a float32), unchanged (a copy) otherwise.
    The norm enters in float64, also where the returned float32 overflows.

    use_norm: a float32 scalar tensor of the same device to use as the norm.
    inplace: write the results into t_list's own tensors (dense, or evenly
    spaced rows; no two may overlap).  None entries stay None.  A NaN norm
    makes every result NaN; an infinite one leaves zeros where the input is finite
    and NaN elsewhere, unless clip_norm is infinite too: then nothing changes."""
    t_list = list(t_list)
    clip_norm = float(clip_norm)
    if not clip_norm >= 0:
        raise ValueError("clip_norm %r is not a number >= 0" % clip_norm)
    l = _List(t_list, inplace)
    if use_norm is not None:
        if _tensor("use_norm", use_norm) != _lib.FP32 or use_norm.numel() != 1 or (
                use_norm.get_device() != l.index):
            raise ValueError("use_norm: expected one float32 on %s" % l.kept[0].device)
        norm, wp, nb, given, to = use_norm, None, 0, use_norm.data_ptr(), None
    else:
        norm, ws, nb = l.empty((), torch.float32), l.empty(l.ws_bytes, torch.uint8), l.ws_bytes
        wp, given, to = ws.data_ptr(), None, norm.data_ptr()
    if inplace:
        out, dst = l.kept, l.ptr
    else:
        out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if l.cols and l.cols[i]
               else torch.empty_like(t) for i, t in enumerate(l.src)]
        dst = array("Q", [t.data_ptr() for t in out])
    _check(lib.ddpg_clip_by_global_norm(
        l.index, _stream(l.index), l.n, l.dtype, l.ptr.buffer_info()[0], dst.buffer_info()[0],
        l.count, *l.rows, clip_norm, given, wp, nb, to))
    if inplace:  # autograd sees the write, as it does torch's own
        torch.autograd.graph.increment_version(out)
    it = iter(out)
    return [None if t is None else next(it) for t in t_list], norm


# ---------------------------------------------------------------- MXFP4
def _mx_bytes(rows, cols):
    return -(-rows // 64) * -(-cols // 128) * 4352


_MX_MAX = 1 << 24  # rows, columns


class MXTensor:
    """A [rows, cols] matrix in MXFP4: 4-bit codes and a scale byte for 32 of
    them along a row, in the order the matrix instructions read (an opaque buffer;
    .dequantize() gives the values).  17/32 byte a value.

    MXTensor(buffer, shape) takes the buffer of another one (a contiguous uint8
    tensor of the shape's size); one on the host is for storage and transport.
    Copies, pickles and torch.save keep (buffer, shape); torch.load reads them with
    torch.serialization.safe_globals([MXTensor])."""

    # the buffer as a view of its own, so that what happens to the caller's tensor
    # (resize_, set_ ..) leaves its size and device; the scales' offset behind the codes
    __slots__ = ("_buffer", "_shape", "_index", "_at")

    def __init__(self, buffer, shape):
        if not isinstance(buffer, torch.Tensor) or buffer.dtype is not torch.uint8 or (
                buffer.layout is not torch.strided):
            raise ValueError("buffer: expected a uint8 tensor, got %s" % (
                buffer.dtype if isinstance(buffer, torch.Tensor) else type(buffer).__name__))
        try:
            rows, cols = (operator.index(n) for n in shape)
        except (TypeError, ValueError):
            raise ValueError("shape: expected (rows, cols), got %r" % (shape,)) from None
        if not (0 <= rows <= _MX_MAX and 0 <= cols <= _MX_MAX):
            raise ValueError("shape: %d x %d is outside [0, %d]" % (rows, cols, _MX_MAX))
        n = _mx_bytes(rows, cols)
        if buffer.numel() != n or not buffer.is_contiguous() or buffer.data_ptr() % 16:
            raise ValueError("buffer: expected %d contiguous bytes, 16-byte aligned, for %d x %d, "
                             "got %s of strides %s" % (n, rows, cols, tuple(buffer.shape),
                                                       buffer.stride()))
        self._set(buffer.view(-1), rows, cols)

    def _set(self, buffer, rows, cols):
        self._buffer, self._shape = buffer, (rows, cols)
        self._index, self._at = buffer.get_device(), buffer.numel() // 17 * 16

    def __reduce__(self):
        return MXTensor, (self._buffer, self._shape)

    buffer = property(lambda self: self._buffer.view(-1))
    shape = property(lambda self: self._shape)

    @property
    def device(self):
        return self._buffer.device

    def dequantize(self, dtype=torch.float32):
        return mx_dequantize(self, dtype)

    def __repr__(self):
        return "MXTensor(%d x %d, %s)" % (*self._shape, self.device)


def _matrix(name, t):
    code = _tensor(name, t)
    if t.dim() != 2:
        raise ValueError("%s: expected [rows, cols], got %s" % (name, tuple(t.shape)))
    return code


def _mx(name, q, cols=None, index=None):
    """(device ordinal, codes, scales) of q."""
    if not isinstance(q, MXTensor):
        raise ValueError("%s: expected an MXTensor (mx_quantize), got %s" % (name,
                                                                            type(q).__name__))
    if cols is not None and q._shape[1] != cols:
        raise ValueError("%s: expected [*, %d], got %s" % (name, cols, q._shape))
    if q._index < 0:
        raise ValueError("%s: expected an MXTensor of the GPU, got one on %s" % (name, q.device))
    if index is not None and q._index != index:
        raise ValueError("%s is on %s, not with the other operands" % (name, q.device))
    codes = q._buffer.data_ptr()  # where it is now: a storage that grows moves
    return q._index, codes, codes + q._at


def mx_quantize(x):
    """x [rows, cols] (float32, bfloat16 or float16, any strides) in MXFP4.

    Blocks of 32 values along a row share the scale 2^(floor(log2(max |x|)) - 2);
    each value becomes the nearest of 0 .5 1 1.5 2 3 4 6 times the scale, ties to
    the even code, larger ones 6.  A block that holds an infinity or a NaN is
    NaN as a whole."""
    code = _matrix("x", x)
    (rows, cols), (s0, s1) = x.shape, x.stride()
    q = object.__new__(MXTensor)
    q._set(x.new_empty(_mx_bytes(rows, cols), dtype=torch.uint8), rows, cols)
    index, codes = q._index, q._buffer.data_ptr()
    _check(lib.ddpg_mx_quantize(index, _stream(index), code, x.data_ptr(), rows, cols, s0, s1,
                                codes, codes + q._at))
    return q


def mx_dequantize(q, dtype=torch.float32):
    """The values q stands for, [rows, cols].  Exact in float32 and bfloat16;
    float16 rounds what lies outside its range."""
    if dtype not in _DTYPES:
        raise ValueError("dtype: %s is none of float32, bfloat16, float16" % dtype)
    index, codes, scales = _mx("q", q)
    rows, cols = q._shape
    out = q._buffer.new_empty((rows, cols), dtype=dtype)
    _check(lib.ddpg_mx_dequantize(index, _stream(index), codes, scales, rows, cols,
                                  _DTYPES[dtype], out.data_ptr(), cols))
    return out


def mx_linear(x, w, bias=None, act=None, dtype=None):
    """act(x w^T + bias), [M, N]: x [M, K] a tensor (quantised on the way) or an
    MXTensor, w [N, K] an MXTensor, bias [N], act None / "elu" / "tanh".  Sums in
    float32; the result is of x's type, or of dtype (float32 if x is an
    MXTensor)."""
    index, w_codes, w_scales = _mx("w", w)
    N, K = w._shape
    wp, nb = None, 0
    if act not in _ACTS:
        raise ValueError("act: %r is none of None, 'elu', 'tanh'" % (act,))
    if isinstance(x, MXTensor):
        _, codes, scales = _mx("x", x, K, index)
        M, xp, xc, s0, s1 = x._shape[0], None, 0, 0, 0
        dtype = dtype or torch.float32
    else:
        xc = _matrix("x", x)
        M, k = x.shape
        if k != K:
            raise ValueError("x: expected [*, %d], got %s" % (K, tuple(x.shape)))
        if x.get_device() != index:
            raise ValueError("x is on %s, w on %s" % (x.device, w.device))
        xp, (s0, s1) = x.data_ptr(), x.stride()
        codes = scales = None
        nb = lib.ddpg_mx_linear_workspace(M, K, N)
        if nb:
            ws = w._buffer.new_empty(nb)
            wp = ws.data_ptr()
        dtype = dtype or x.dtype
    yc = _DTYPES.get(dtype)
    if yc is None:
        raise ValueError("dtype: %s is none of float32, bfloat16, float16" % dtype)
    bc, bp = 0, None
    if bias is not None:
        bc = _tensor("bias", bias)
        if bias.shape != (N,) or bias.get_device() != index:
            raise ValueError("bias: expected [%d] on %s, got %s on %s" % (
                N, w.device, tuple(bias.shape), bias.device))
        bias = bias.contiguous()
        bp = bias.data_ptr()
    y = w._buffer.new_empty((M, N), dtype=dtype)
    _check(lib.ddpg_mx_linear(index, _stream(index), xc, xp, s0, s1, codes, scales, M, K, w_codes,
                              w_scales, N, bc, bp, _ACTS[act], yc, y.data_ptr(), N, wp, nb))
    return y


def mx_linear_grad(dy, x, w, need=(True, True), bias=True):
    """(dx, dw, db) of mx_linear's product x w^T + bias (before act) for dy
    [M, N], with the values the MXTensors x [M, K] and w [N, K] stand for: dx = dy w
    of dy's type, dw = dy^T x and db = dy's column sums in float32.  dy may have any
    strides; adjacent columns are read fastest.  The quantisation's own derivative is
    taken as 1 (straight-through), so dx and dw are the gradients of the matrices that
    were quantised.  need: whether dx, dw are wanted (None otherwise); bias:
    whether db is."""
    code = _matrix("dy", dy)
    index = dy.get_device()
    _, x_codes, x_scales = _mx("x", x, None, index)
    M, K = x._shape
    _, w_codes, w_scales = _mx("w", w, K, index)
    N = w._shape[0]
    if dy.shape != (M, N):
        raise ValueError("dy: expected [%d, %d], got %s" % (M, N, tuple(dy.shape)))
    dx = dw = db = pdx = pdw = pdb = None
    if need[0]:
        dx = dy.new_empty((M, K))
        pdx = dx.data_ptr()
    if need[1]:
        dw = dy.new_empty((N, K), dtype=torch.float32)
        pdw = dw.data_ptr()
    if bias:
        db = dy.new_empty(N, dtype=torch.float32)
        pdb = db.data_ptr()
    nb = lib.ddpg_mx_linear_grad_workspace(code, M, N, K, dx is not None, dw is not None,
                                           db is not None)
    ws = x._buffer.new_empty(nb)
    s0, s1 = dy.stride()
    _check(lib.ddpg_mx_linear_grad(index, _stream(index), code, dy.data_ptr(), s0, s1, M, N, K,
                                   x_codes, x_scales, w_codes, w_scales, pdx, pdw, pdb,
                                   ws.data_ptr(), nb))
    return dx, dw, db
