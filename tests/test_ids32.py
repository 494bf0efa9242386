"""64-bit ids and lengths narrowed for the kernels: values outside the range stay outside."""
import pytest
import torch

from fastest_flash_attention_b200 import _lib
from fastest_flash_attention_b200.kv_cache import _id_pair


@pytest.mark.parametrize("limit", [1, 8, 2 ** 31 - 1])
def test_values_outside_stay_outside(limit):
    x = torch.tensor([0, limit - 1, -1, limit, limit + 5, 2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 63 - 1, -2 ** 63])
    got = _lib.int32(x, limit)
    assert got.dtype == torch.int32 and got[:2].tolist() == [0, limit - 1]
    assert bool(((got[2:] < 0) | (got[2:] >= limit)).all())
    small = torch.arange(8, dtype=torch.int32)
    assert _lib.int32(small) is small and _lib.int32(small[::2]).tolist() == [0, 2, 4, 6]


def test_pools_past_32_bit_ids():
    ids = torch.tensor([1]), torch.tensor([2])
    with pytest.raises(ValueError, match="32-bit"):
        _id_pair(*ids, 2 ** 31, torch.device("cpu"), "slot")
    pair = _id_pair(*(t.int() for t in ids), 2 ** 31, torch.device("cpu"), "slot")
    assert [t.tolist() for t in pair] == [[1], [2]]
