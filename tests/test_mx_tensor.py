"""MXTensor as an object (no GPU needed): what its constructor and the operators
refuse, and that a copy stands on its own buffer."""
import copy
import io
import pickle

import pytest
import torch

from distributed_ddpg_amd import ops

TILE = 4352  # bytes of 64 rows x 128 columns: 4096 of codes, 256 of scales


def make(rows=8, cols=4, n=TILE):
    return ops.MXTensor(torch.arange(n, dtype=torch.int32).to(torch.uint8), (rows, cols))


def through_torch(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    with torch.serialization.safe_globals([ops.MXTensor]):
        return torch.load(f, weights_only=True)


COPIES = {"deepcopy": copy.deepcopy, "pickle": lambda q: pickle.loads(pickle.dumps(q)),
          "torch.save": through_torch}


@pytest.mark.parametrize("how", sorted(COPIES))
def test_a_copy_has_its_own_buffer(how):
    q = make(65, 129, 4 * TILE)
    c = COPIES[how](q)
    assert c.shape == q.shape == (65, 129) and torch.equal(c.buffer, q.buffer)
    assert c.buffer.data_ptr() != q.buffer.data_ptr()
    kept = c.buffer.clone()
    q.buffer.zero_()
    assert torch.equal(c.buffer, kept)
    held = [getattr(c, slot) for slot in q.__slots__]  # nothing that names the old memory
    assert not [v for v in held if isinstance(v, int) and v >= q.buffer.data_ptr()]


def test_a_shallow_copy_shares_it():
    q = make()
    s = copy.copy(q)
    q.buffer.fill_(7)
    assert s.buffer.data_ptr() == q.buffer.data_ptr() and (s.buffer == 7).all()


def test_the_shape_and_the_buffer_are_fixed():
    q = make()
    with pytest.raises(AttributeError):
        q.shape = (100000, 100000)
    with pytest.raises(AttributeError):
        q.buffer = torch.empty(0, dtype=torch.uint8)


u8 = torch.uint8


@pytest.mark.parametrize("buffer,shape", [
    (torch.empty(TILE, dtype=u8), (100000, 100000)),          # too small
    (torch.empty(2 * TILE, dtype=u8), (64, 128)),             # too large
    (torch.empty(TILE, dtype=u8), (65, 128)),
    (torch.empty(TILE, dtype=u8), (64, 129)),
    (torch.empty(TILE, dtype=torch.int8), (64, 128)),
    (torch.empty(TILE // 4, dtype=torch.float32), (64, 128)),
    (torch.empty(2 * TILE, dtype=u8)[::2], (64, 128)),        # not contiguous
    (torch.empty(1, dtype=u8).expand(TILE), (64, 128)),
    (torch.empty(TILE + 16, dtype=u8)[1:TILE + 1], (64, 128)),  # not 16-byte aligned
    (None, (64, 128)),
    (torch.empty(TILE, dtype=u8), (64,)),
    (torch.empty(TILE, dtype=u8), (64, 128, 1)),
    (torch.empty(TILE, dtype=u8), (-64, -128)),
    (torch.empty(TILE, dtype=u8), (64.0, 128)),
    (torch.empty(TILE, dtype=u8), 64),
    (torch.empty(0, dtype=u8), ((1 << 24) + 1, 0)),
])
def test_the_constructor_refuses(buffer, shape):
    with pytest.raises(ValueError):
        ops.MXTensor(buffer, shape)


def test_what_it_takes():
    assert ops.MXTensor(torch.empty(0, dtype=u8), (0, 40)).shape == (0, 40)
    assert ops.MXTensor(torch.empty(TILE, dtype=u8), torch.Size([64, 128])).shape == (64, 128)
    assert ops.MXTensor(torch.empty(1, TILE, dtype=u8), [1, 1]).shape == (1, 1)


def test_the_operators_refuse_one_on_the_host():
    q = make()
    for f in (lambda: q.dequantize(), lambda: ops.mx_linear(q, q),
              lambda: ops.mx_linear(q, q, dtype=torch.float16)):
        with pytest.raises(ValueError, match="cpu"):
            f()


@pytest.mark.parametrize("cut", [lambda b: b.resize_(16), lambda b: b.resize_(0),
                                 lambda b: b.set_(torch.empty(17, dtype=u8)),
                                 lambda b: b.as_strided_((TILE,), (0,)),
                                 lambda b: b.resize_(1 << 20)])
@pytest.mark.parametrize("whose", ["the caller's", "the handed out"])
def test_it_stays_whole_when_a_buffer_changes(cut, whose):
    mine = torch.arange(TILE, dtype=torch.int32).to(u8)
    want = mine.clone()
    q = ops.MXTensor(mine, (8, 4))
    cut(mine if whose == "the caller's" else q.buffer)
    assert q.buffer.shape == (TILE,) and q.buffer.stride() == (1,) and torch.equal(q.buffer, want)
