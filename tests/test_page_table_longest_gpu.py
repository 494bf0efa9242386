"""A slot map of nearly 2^31 places: positions past 2^31 - 65536, where a warp's next step would pass 2^31."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [2 ** 31 - 1, 2 ** 31 - 65536])
def test_largest_slot_map(tokens):
    from fastest_flash_attention_b200 import assign_slots

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    bt, ring, state = ints([[-1, -1], [-1, -1]]), ints([3, 1, 2, 0]), ints([0, 4])
    guard = [torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda") for _ in range(4)]
    plan = assign_slots(bt, ints([0, 0]), ints([5, 17]), ring, state, page_size=16, max_tokens=tokens)
    assert plan.starts.tolist() == [0, 5, 22] and plan.free_state.tolist() == [3, 1]
    assert bt.tolist() == [[3, -1], [1, 2]]
    assert plan.slots[:22].tolist() == [48 + i for i in range(5)] + [16 + i for i in range(16)] + [32]
    assert plan.positions[:22].tolist() == list(range(5)) + list(range(17))
    for at in range(22, tokens, 1 << 28):
        assert bool((plan.slots[at:at + (1 << 28)] == -1).all()) and bool((plan.positions[at:at + (1 << 28)] == 0).all())
    assert all(bool((g == 7).all()) for g in guard)
