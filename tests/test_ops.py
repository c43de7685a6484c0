"""What the tensor operators refuse (no GPU needed: every check comes before
the first device call), and their oracle's own values."""
import ctypes

import pytest
import torch

from distributed_ddpg_amd import _lib, ops
from oracle import ops_oracle as O

L = _lib.lib


def refused(rc, *words):
    msg = L.ddpg_global_error().decode()
    assert rc == _lib.DDPG_EINVAL, (rc, msg)
    assert all(w in msg for w in words), msg


def test_python_refusals():
    cpu = torch.zeros(4, 4)
    for f in (lambda: ops.global_norm([cpu]), lambda: ops.global_norm([]),
              lambda: ops.global_norm([None]), lambda: ops.global_norm([3.0]),
              lambda: ops.clip_by_global_norm([cpu], 1.0),
              lambda: ops.clip_by_global_norm([cpu], -1.0),
              lambda: ops.clip_by_global_norm([cpu], float("nan")),
              lambda: ops.mx_quantize(cpu), lambda: ops.mx_dequantize(cpu),
              lambda: ops.mx_linear(cpu, cpu), lambda: ops.mx_linear_grad(cpu, cpu, cpu)):
        with pytest.raises(ValueError):
            f()
    buf = torch.empty(4352, dtype=torch.uint8)
    q = ops.MXTensor(buf, (8, 4))
    with pytest.raises(ValueError):
        ops.mx_dequantize(q, torch.float64)
    with pytest.raises(ValueError):
        ops.mx_linear(cpu, q, act="relu")
    with pytest.raises(ValueError):
        ops.mx_linear(ops.MXTensor(buf, (3, 5)), q)


def arr(t, *v):
    return (t * len(v))(*v)


def test_norm_entry_refusals():
    one, p = arr(ctypes.c_int64, 8), arr(ctypes.c_void_p, 4096)
    f32, bad = arr(ctypes.c_int, 0), arr(ctypes.c_int, 7)
    norm = lambda *a: L.ddpg_global_norm(0, None, *a)
    refused(norm(-1, f32, p, one, None, None, 1, 1 << 20, 1), "length")
    refused(norm(1, bad, p, one, None, None, 1, 1 << 20, 1), "dtype 7")
    refused(norm(1, None, p, one, None, None, 1, 1 << 20, 1), "null")
    refused(norm(1, f32, arr(ctypes.c_void_p, 0), one, None, None, 1, 1 << 20, 1), "null")
    refused(norm(1, f32, p, arr(ctypes.c_int64, -1), None, None, 1, 1 << 20, 1), "-1 elements")
    refused(norm(1, f32, p, one, one, None, 1, 1 << 20, 1), "together")
    refused(norm(1, f32, p, one, arr(ctypes.c_int64, 3), one, 1, 1 << 20, 1), "rows of 3")
    refused(norm(1, f32, p, one, None, None, None, 0, 1), "null")
    refused(norm(1, f32, p, one, None, None, 1, 1 << 20, None), "null")
    clip = lambda c, n=1, src=p, dst=p, cnt=one, cols=None, ld=None: L.ddpg_clip_by_global_norm(
        0, None, n, arr(ctypes.c_int, *[0] * n), src, dst, cnt, cols, ld, c, None, 1, 1 << 20, 1)
    refused(clip(-1.0), "clip_norm")
    refused(clip(float("nan")), "clip_norm")
    two = arr(ctypes.c_int64, 8, 8)
    at = arr(ctypes.c_void_p, 4096, 4096 + 28)
    refused(clip(1.0, 2, at, at, two), "tensors 0 and 1 overlap")
    twice = arr(ctypes.c_void_p, 4096, 4096)
    refused(clip(1.0, 2, twice, twice, two), "tensors 0 and 1 overlap")
    refused(clip(1.0, 1, p, p, one, arr(ctypes.c_int64, 4), arr(ctypes.c_int64, 3)), "itself")
    refused(L.ddpg_clip_by_global_norm(0, None, 1, f32, p, p, one, None, None, 1.0, 4100, None, 0,
                                       None), "use_norm lies in tensor 0")
    # two column ranges of rows 10 apart that share column 3
    cols, ld = arr(ctypes.c_int64, 4, 4), arr(ctypes.c_int64, 10, 10)
    at = arr(ctypes.c_void_p, 4096, 4096 + 3 * 4)
    refused(clip(1.0, 2, at, at, two, cols, ld), "overlap")


def test_single_rows_without_a_pitch():
    """A single row may name any distance to the next, 0 too."""
    dt, n = arr(ctypes.c_int, 0, 0), arr(ctypes.c_int64, 8, 8)
    at = arr(ctypes.c_void_p, 4096, 4096 + 16)
    for pitch in (0, 4, 1 << 56):
        ld = arr(ctypes.c_int64, pitch, pitch)
        refused(L.ddpg_clip_by_global_norm(0, None, 2, dt, at, at, n, n, ld, 1.0, None, 1, 1 << 20,
                                           1), "tensors 0 and 1 overlap")
    ld = arr(ctypes.c_int64, 1 << 56, 1 << 56)  # two rows: their span leaves 64 bits
    refused(L.ddpg_clip_by_global_norm(0, None, 2, dt, at, at, n, arr(ctypes.c_int64, 4, 4), ld, 1.0,
                                       None, 1, 1 << 20, 1), "rows of 4")


def test_learner_clip_values():
    from distributed_ddpg_amd.networks import _clip_norm
    assert [_clip_norm(x) for x in (None, 2, 2.0 ** -149, float("inf"))] == [
        0.0, 2.0, 2.0 ** -149, float("inf")]
    for bad in (0, -1.0, float("nan"), 1e-50):  # 1e-50 is 0, no clip, in float32
        with pytest.raises(ValueError):
            _clip_norm(bad)


def test_mx_entry_refusals():
    big = (1 << 24) + 1
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    refused(L.ddpg_mx_sizes(-1, 4, a, b), "-1 x 4")
    refused(L.ddpg_mx_sizes(4, big, a, b), "outside")
    assert L.ddpg_mx_sizes(65, 129, a, b) == 0 and (a.value, b.value) == (4 * 4096, 4 * 256)
    refused(L.ddpg_mx_quantize(0, None, 9, 16, 4, 4, 4, 1, 16, 16), "dtype 9")
    refused(L.ddpg_mx_quantize(0, None, 0, None, 4, 4, 4, 1, 16, 16), "null")
    refused(L.ddpg_mx_quantize(0, None, 0, 16, 4, 4, 4, 1, None, 16), "null")
    refused(L.ddpg_mx_quantize(0, None, 0, 16, 4, 4, 4, 1, 24, 16), "aligned")
    refused(L.ddpg_mx_quantize(0, None, 0, 16, big, 4, 4, 1, 16, 16), "outside")
    refused(L.ddpg_mx_dequantize(0, None, 16, 16, 4, 4, 0, 16, 3), "overlap")
    refused(L.ddpg_mx_dequantize(0, None, 16, 16, 4, 4, 5, 16, 4), "dtype 5")
    lin = lambda **k: L.ddpg_mx_linear(0, None, k.get("xd", 0), k.get("x"), 4, 1, 16, 16,
                                       k.get("M", 4), k.get("K", 4), k.get("w", 16), 16, 4,
                                       k.get("bd", 0), k.get("b"), k.get("act", 0),
                                       k.get("dt", 0), k.get("y", 16), k.get("ld", 4),
                                       k.get("ws"), k.get("nb", 0))
    refused(lin(M=-1), "outside")
    refused(lin(K=big), "outside")
    refused(lin(w=None), "null")
    refused(lin(act=3), "act 3")
    refused(lin(dt=4), "dtype 4")
    refused(lin(x=16, xd=4), "dtype 4")
    refused(lin(b=16, bd=4), "dtype 4")
    refused(lin(y=None), "null")
    refused(lin(ld=3), "overlap")
    refused(lin(M=100, x=16), "workspace")
    nb = L.ddpg_mx_linear_workspace(100, 4, 4)
    assert nb == 2 * 4352 and L.ddpg_mx_linear_workspace(1, 4, 4) == 0
    refused(lin(M=100, x=16, ws=24, nb=nb), "workspace")
    need = L.ddpg_mx_linear_grad_workspace(0, 4, 4, 4, 1, 1, 1)
    assert need > 0 and L.ddpg_mx_linear_grad_workspace(0, 4, 4, 4, 0, 0, 0) == 0
    grad = lambda **k: L.ddpg_mx_linear_grad(0, None, k.get("dt", 0), k.get("dy", 16), 4, 1,
                                             k.get("M", 4), 4, 4, k.get("x", 16), 16,
                                             k.get("w", 16), 16, 16, 16, 16, k.get("ws", 256),
                                             k.get("nb", need))
    refused(grad(dt=3), "dtype 3")
    refused(grad(dy=None), "null")
    refused(grad(x=None), "null")
    refused(grad(w=None), "null")
    refused(grad(nb=need - 1), "workspace")
    refused(grad(ws=None), "workspace")
    refused(grad(M=-4), "outside")


def test_oracle_values_by_hand():
    x = torch.tensor([[7.0, 5.0, 2.5, -3.5, 0.25, 0.75, 1.25, 1.75] + [0.0] * 24])
    assert O.mx_values(x)[0, :8].tolist() == [6.0, 4.0, 2.0, -4.0, 0.0, 1.0, 1.0, 2.0]
    y = torch.tensor([[0.3] + [0.01] * 31])  # E = floor(log2 0.3) - 2 = -4
    assert O.mx_values(y)[0, :2].tolist() == [4.0 / 16, 0.0]
