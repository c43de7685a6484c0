"""Tensor lists that mix tensors clipped in place with others, and their rows (no GPU
needed: the checks come first; a call that passes them ends at a device that is not
there)."""
import ctypes

import pytest
import torch

from distributed_ddpg_amd import _lib, ops

L = _lib.lib
NO_DEVICE = 99
FAR = 1 << 40


def arr(t, v):
    return (t * len(v))(*v)


def clip(tensors):
    """rc of a clip of [(src, dst, count, cols, ld)] of float32."""
    src, dst, count, cols, ld = zip(*tensors)
    return L.ddpg_clip_by_global_norm(
        NO_DEVICE, None, len(tensors), arr(ctypes.c_int, [0] * len(src)),
        arr(ctypes.c_void_p, src), arr(ctypes.c_void_p, dst), arr(ctypes.c_int64, count),
        arr(ctypes.c_int64, cols), arr(ctypes.c_int64, ld), 1.0, None, 16, 1 << 20, 16)


INPLACE = (FAR, FAR, 8, 0, 0)


@pytest.mark.parametrize("other", [
    (FAR + 4096, FAR + 8192, 32, 8, 0),         # a broadcast row, written dense
    (FAR + 4096, FAR + 8192, 32, 8, 5),         # rows that share elements
    (FAR + 4096, FAR - 128, 32, 8, 1 << 20),    # dense results right before, rows far apart
    (FAR + 4096, FAR + 32, 8, 1, 1 << 10),      # .. and right behind
])
def test_a_tensor_of_its_own_destination_is_dense_there(other):
    for tensors in ([INPLACE, other], [other, INPLACE]):
        assert clip(tensors) == _lib.DDPG_EHIP, L.ddpg_global_error()


@pytest.mark.parametrize("other", [
    (FAR + 4096, FAR + 28, 8, 0, 0),            # its results on the last element
    (FAR + 4096, FAR - 124, 32, 8, 1 << 20),
    (FAR + 28, FAR + 4096, 8, 0, 0),            # its input: read while the other is written
    (FAR - 1024 * 4, FAR + 4096, 32, 8, 256),   # rows, the last of them before it ..
    (FAR - 1024 * 4, FAR + 4096, 40, 8, 256),   # .. and one on it
])
def test_what_meets_is_refused(other):
    meets = other[:1] != (FAR - 1024 * 4,) or other[2] == 40
    for tensors in ([INPLACE, other], [other, INPLACE]):
        rc = clip(tensors)
        assert rc == (_lib.DDPG_EINVAL if meets else _lib.DDPG_EHIP), L.ddpg_global_error()
        if meets:
            assert b"overlap" in L.ddpg_global_error()


def test_rows_longer_than_the_kernels_count():
    """Such rows go through a dense copy (a meta tensor: nothing is allocated)."""
    t = torch.empty(2, (1 << 31) + 8, device="meta")
    assert ops._rows(t[:, :1 << 31]) is None
    assert ops._rows(t[:, :(1 << 31) - 1]) == ((1 << 31) - 1, (1 << 31) + 8)
