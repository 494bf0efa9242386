"""Which neighbouring sequences of a host cache decode as one group."""
import pytest
import torch

import fastest_flash_attention_b200 as ffa


def _cache():
    return ffa.PagedKVCache(max_pages=64, page_size=4, num_heads=1, head_dim=4, dtype=torch.float32)


def _add(c, s, n):
    x = torch.zeros(1, n, 4)
    c.append_tokens(s, x, x)


def test_forks_are_a_group():
    c = _cache()
    _add(c, "a", 10)
    c.fork_sequences([("a", "b"), ("a", "c")])
    for s, n in (("b", 7), ("c", 1)):
        _add(c, s, n)
    _add(c, "x", 9)
    assert c.prefix_groups(["a", "b", "c", "x"]) == ([0, 3, 4], [8, 0])
    assert c.prefix_groups(["x", "b", "c"]) == ([0, 1, 3], [0, 8])
    assert c.prefix_groups(["a", "x", "b"]) == ([0, 1, 2, 3], [0, 0, 0])  # neighbours alone
    assert c.prefix_groups(["x"]) == ([0, 1], [0])
    c.fork_sequence("b", "d")  # 17 tokens: 16 in common with b, 8 with a
    _add(c, "d", 3)
    assert c.prefix_groups(["b", "d"]) == ([0, 2], [16])
    assert c.prefix_groups(["b", "d", "a"]) == ([0, 3], [8])   # 8 + 8 saved against 16
    _add(c, "b", 20)
    c.fork_sequence("b", "e")  # 36 in common with b
    assert c.prefix_groups(["b", "e", "a"]) == ([0, 2, 3], [36, 0])  # a would cost 28 and bring 8


def test_short_sequences_and_no_full_page():
    c = _cache()
    _add(c, "a", 3)
    c.fork_sequence("a", "b")
    assert c.prefix_groups(["a", "b"]) == ([0, 1, 2], [0, 0])
    _add(c, "z", 0)
    assert c.prefix_groups(["z", "a"]) == ([0, 1, 2], [0, 0])


def test_refusals():
    c = _cache()
    _add(c, "a", 8)
    q = torch.zeros(1, 1, 4)
    with pytest.raises(ValueError):
        c.decode(q, ["a"], share_prefix=True, sliding_window=4)
    for ids, new in ((["a"], [2]), (["a"], [1, 0]), (["a"], [9])):
        with pytest.raises(ValueError):
            c.prefill(q if new != [9] else torch.zeros(9, 1, 4), ids, new)
