"""Operands on different GPUs are refused before any pointer reaches a kernel.
No GPU: the tensors here have a device and a shape but no memory."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fastest_flash_attention_b200 as ffa
from fastest_flash_attention_b200 import attention


@pytest.fixture
def empty():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.bfloat16, on=0: torch.empty(*shape, dtype=dtype, device=f"cuda:{on}")


def _each_moved(call, args, movable):
    """Calls with one operand at a time on the other GPU."""
    for i in movable:
        moved = [a.to("cuda:1") if j == i else a for j, a in enumerate(args)]
        with pytest.raises(ValueError, match="one device"):
            call(*moved)


def test_attention(empty):
    q, k, v = (empty(1, 2, 8, 64) for _ in range(3))
    _each_moved(lambda *a: attention.flash_fwd(*a, scale=1.0, window=4, sink=1), [q, k, v], range(3))
    lse = empty(1, 2, 8, dtype=torch.float32)
    _each_moved(lambda *a: attention.flash_bwd(*a, scale=1.0, window=4, sink=1), [q, q, k, v, q, lse], range(6))


def test_paged_decode(empty):
    args = [empty(2, 4, 64), empty(6, 2, 16, 64), empty(6, 2, 16, 64), empty(2, 3, dtype=torch.int32),
            empty(2, dtype=torch.int32)]
    for kw in (dict(sliding_window=8, sink_tokens=2), dict()):
        _each_moved(lambda *a: ffa.paged_decode(*a, **kw), args, range(5))


def test_rotary(empty):
    q, k, cos, sin = empty(1, 2, 8, 64), empty(1, 1, 8, 64), *(empty(32, 32, dtype=torch.float32) for _ in range(2))
    pos = empty(8, dtype=torch.int32)
    _each_moved(ffa.apply_rotary, [q, k, cos, sin, pos], range(5))
    args = [empty(8, 2, 64), empty(8, 1, 64), empty(8, 1, 64), cos, sin, pos, pos, empty(4, 1, 16, 64), empty(4, 1, 16, 64)]
    _each_moved(ffa.rotary_append, args, range(9))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_copies(empty, dtype):
    """Page ids and slots are brought to the pool's GPU, whichever they are on; the pools themselves are not moved."""
    from fastest_flash_attention_b200.kv_cache import _id_pair
    for a, b in ((0, 0), (0, 1), (1, 0), (1, 1)):
        pair = _id_pair(empty(2, dtype=dtype, on=a), empty(2, dtype=dtype, on=b), 4, torch.device("cuda:0"), "page id")
        assert [(t.device.index, t.dtype) for t in pair] == [(0, torch.int32)] * 2
    ids = empty(2, dtype=dtype)
    for fn in (ffa.copy_pages, ffa.move_tokens):
        _each_moved(lambda k, v: fn(k, v, ids, ids), [empty(4, 1, 16, 64), empty(4, 1, 16, 64)], range(2))
