"""Refusals of the page-table calls that need no GPU."""
import pytest
import torch

import fastest_flash_attention_b200 as ffa


def test_entry_points_refuse_sizes_that_mean_nothing():
    from fastest_flash_attention_b200 import _lib
    lib, p = _lib.load(), 4096  # never dereferenced: the sizes are refused first
    bad = (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
    for width, R, P, page, tokens in ((0, 1, 4, 16, 1), (4, -1, 4, 16, 1), (4, 1, 0, 16, 1), (4, 1, 4, 0, 1),
                                      (4, 1, 4, 16, -1), (4, 16385, 4, 16, 1), (4, 1, 2 ** 30, 16, 1),
                                      (2 ** 30, 1, 4, 16, 1)):
        assert lib.ffa_assign_slots(p, width, p, p, p, p, p, p, p, p, p, R, P, page, tokens, None, None) in bad
        if tokens > 0:
            assert lib.ffa_release_pages(p, width, p, p, None, p, p, p, p, R, P, page, None, None) in bad
    args = [p, 4, p, p, p, p, p, p, p, p, p, 1, 4, 16, 1, None, None]
    for i in (0, 2, 3, 4, 5, 6, 7, 8, 9, 10):
        assert lib.ffa_assign_slots(*args[:i], None, *args[i + 1:]) == _lib.FFA_ERR_INVALID_ARG
    args = [p, 4, p, p, None, p, p, p, p, 1, 4, 16, None, None]
    for i in (0, 2, 3, 5, 6, 7, 8):
        assert lib.ffa_release_pages(*args[:i], None, *args[i + 1:]) == _lib.FFA_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.assign_slots(z[None], z, z, z, z.repeat(2), page_size=16, max_tokens=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.release_pages(z[None], z, z.bool(), z, z.repeat(2), page_size=16)
    t = ffa.DevicePageTable(2, 4, 8, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        t.assign(torch.ones(2, dtype=torch.int32), 2)
    for sizes in ((0, 4, 8), (2, 0, 8), (2, 4, 0)):
        with pytest.raises(ValueError):
            ffa.DevicePageTable(*sizes, device="cpu")


def _meta(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype)


def test_shapes_and_types_are_refused(monkeypatch):
    """The checks behind the device's, on host tensors."""
    from fastest_flash_attention_b200 import _lib
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", lambda: pytest.fail("the call was not refused"))
    good = dict(bt=_meta(2, 4), lens=_meta(2), rows=_meta(2), ring=_meta(8), state=_meta(2))
    for change in (dict(bt=_meta(4)), dict(bt=_meta(2, 0)), dict(bt=_meta(2, 4, dtype=torch.int64)),
                   dict(bt=_meta(4, 2).t()), dict(lens=_meta(3)), dict(lens=_meta(2, dtype=torch.int64)),
                   dict(lens=_meta(4)[::2]), dict(rows=_meta(3)), dict(rows=_meta(2, dtype=torch.float32)),
                   dict(ring=_meta(0)), dict(ring=_meta(8, dtype=torch.int64)), dict(state=_meta(3)),
                   dict(state=_meta(2, dtype=torch.int64))):
        a = dict(good, **change)
        with pytest.raises(ValueError):
            ffa.assign_slots(a["bt"], a["lens"], a["rows"], a["ring"], a["state"], page_size=16, max_tokens=4)
        done = a["rows"] if a["rows"].dtype is torch.float32 else a["rows"].bool()
        with pytest.raises(ValueError):
            ffa.release_pages(a["bt"], a["lens"], done, a["ring"], a["state"], page_size=16)
    args = (good["bt"], good["lens"], good["rows"], good["ring"], good["state"])
    for kw in (dict(page_size=0, max_tokens=1), dict(page_size=16, max_tokens=-1)):
        with pytest.raises(ValueError):
            ffa.assign_slots(*args, **kw)
    for keep in (_meta(3), _meta(2, dtype=torch.float32)):
        with pytest.raises(ValueError):
            ffa.release_pages(good["bt"], good["lens"], good["rows"].bool(), good["ring"], good["state"], page_size=16,
                              keep=keep)
