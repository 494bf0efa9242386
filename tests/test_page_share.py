"""Refusals of sharing a prefix that need no GPU."""
import ctypes

import pytest
import torch

import fastest_flash_attention_b200 as ffa


def test_entry_point_refuses_what_means_nothing():
    from fastest_flash_attention_b200 import _lib
    lib, p = _lib.load(), 4096  # never dereferenced: the arguments are refused first
    bad = (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)

    def call(table=p, width=4, lens=p, owner=0, rows=(1, 2), R=4, P=8, page=16, tokens=32, n=None):
        ids = (ctypes.c_int * len(rows))(*rows) if rows is not None else None
        return lib.ffa_share_pages(table, width, lens, owner, ids, len(rows) if n is None else n, R, P, page, tokens,
                                   None, None)
    for kw in (dict(table=None), dict(lens=None), dict(width=0), dict(owner=-1), dict(owner=4), dict(rows=(1, 1)),
               dict(rows=(0,)), dict(rows=(4,)), dict(rows=(-1,)), dict(rows=None, n=1), dict(n=-1), dict(R=0),
               dict(R=-1), dict(R=16385), dict(P=0), dict(P=2 ** 30), dict(page=0), dict(tokens=0), dict(tokens=-16),
               dict(tokens=17), dict(tokens=80), dict(width=2 ** 30)):
        assert call(**kw) in bad, kw
    assert call(rows=()) == _lib.FFA_OK


def test_arguments_are_refused(monkeypatch):
    from fastest_flash_attention_b200 import _lib
    t = ffa.DevicePageTable(4, 8, 20, page_size=16, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        t.share(0, [1], 16)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("the call was not refused"))
    for owner, rows, tokens in ((0, [1], 5), (0, [1], 0), (0, [1], -16), (0, [0], 16), (0, [1, 1], 16), (0, [4], 16),
                                (4, [1], 16), (-1, [1], 16), (0, [-1], 16), (0, [1], 16 * 9)):
        with pytest.raises(ValueError):
            t.share(owner, rows, tokens)
    t.ctx_lens = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        t.share(0, [1], 16)
