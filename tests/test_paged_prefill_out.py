"""Which layouts of ``out`` paged_prefill takes: those whose heads share no memory, found here by counting."""
import itertools

import pytest
import torch

import fastest_flash_attention_b200 as ffa


def _overlaps(T, H, D, st, sh):
    at = torch.tensor([t * st + h * sh + d for t in range(T) for h in range(H) for d in range(D)])
    return at.unique().numel() < at.numel()


def test_heads_that_overlap_are_refused_and_no_others(monkeypatch):
    from fastest_flash_attention_b200 import _lib

    class Reached(Exception):
        pass

    class Stub:
        def ffa_paged_prefill(self, *args):
            raise Reached
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", Stub)
    monkeypatch.setattr(_lib, "err_ptr", lambda t: 0)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "device_of", lambda t: _lib._HERE)
    D = 16
    strides = [0, 8, 16, 24, 32, 40, 48, 64, 80, 128]
    seen = set()
    for T, H, st, sh in itertools.product((1, 2, 4, 5), (1, 2, 3, 8), strides, strides):
        q, pool = torch.zeros(T, H, D).half(), torch.zeros(3, 1, 16, D).half()
        out = torch.zeros(T * st + H * sh + D).half()
        out = out[-out.data_ptr() % 16 // 2:].as_strided((T, H, D), (st, sh, 1))
        bad = _overlaps(T, H, D, st, sh)
        seen.add(bad)
        with pytest.raises(ValueError if bad else Reached):
            ffa.paged_prefill(q, pool, pool, torch.zeros(1, 3).int(), torch.zeros(1).int(), torch.zeros(2).int(),
                              out=out)
    assert seen == {True, False}


@pytest.mark.parametrize("strides", [(64, 64, 1), (128, 64, 1), (64, 192, 1)])
def test_tokens_that_lie_in_each_other_are_refused(strides, monkeypatch):
    from fastest_flash_attention_b200 import _lib
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", lambda: pytest.fail("the call was not refused"))
    pool = torch.zeros(3, 2, 16, 64).half()
    out = torch.zeros(4096).half()
    out = out[-out.data_ptr() % 16 // 2:].as_strided((4, 8, 64), strides)
    with pytest.raises(ValueError, match="apart"):
        ffa.paged_prefill(torch.zeros(4, 8, 64).half(), pool, pool, torch.zeros(2, 3).int(), torch.zeros(2).int(),
                          torch.zeros(3).int(), out=out)
