"""Host side of the streaming operators where a call is refused or its inputs
change between calls: what a failing call leaves behind, and what arguments
may be.  No GPU: host-side pools, stand-ins for the launches, or tensors that
have a device but no memory."""
import pytest
import torch

import fastest_flash_attention_b200 as ffa


def _cache(pages=8, ps=4):
    return ffa.PagedKVCache(max_pages=pages, page_size=ps, num_heads=2, head_dim=4, dtype=torch.float32)


def _tokens(n, base=0):
    k = (torch.arange(n, dtype=torch.float32) + base)[None, :, None].expand(2, n, 4).contiguous()
    return k, -k


def test_append_without_enough_pages_changes_nothing():
    c = _cache(pages=3)
    with pytest.raises(RuntimeError, match="out of physical pages"):
        c.append_tokens(0, *_tokens(13))
    assert not c.sequences and c.free_pages == [0, 1, 2]
    c.append_tokens(0, *_tokens(5))
    with pytest.raises(RuntimeError, match="out of physical pages"):
        c.append_tokens(0, *_tokens(8, 5))
    assert c.sequences[0]["len"] == 5 and c.sequences[0]["page_table"] == [0, 1] and c.free_pages == [2]
    c.append_tokens(0, *_tokens(7, 5))  # what fits still does
    assert c.get_kv(0)[0][0, :, 0].tolist() == list(range(12))
