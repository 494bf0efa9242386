"""Numbers of any type that converts to the parameter's reach the library's
entry points (no GPU: the library is replaced by its signatures)."""
import contextlib

import numpy as np
import pytest
import torch

from fastest_flash_attention_b200 import _lib, attention


class _Signatures:
    """Stands for the library: converts every argument as ctypes does and keeps what the last call got."""

    def __getattr__(self, name):
        def call(*args):
            types = _lib.SIGNATURES[name][1]
            assert len(args) == len(types), name
            for a, t in zip(args, types):
                if not isinstance(a, tuple):
                    t.from_param(a)
            self.last = name, args
            return 1 << 10 if "workspace_size" in name else _lib.FFA_OK
        return call


@pytest.fixture
def lib(monkeypatch):
    lib = _Signatures()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "direct", lambda: lib)
    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "err_ptr", lambda t: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: None)
    monkeypatch.setattr(_lib, "sync_check_enabled", lambda: False)
    attention._sink_workspace.cache_clear()
    yield lib
    attention._sink_workspace.cache_clear()


def _qkv():
    return tuple(torch.zeros(1, 2, 32, 64, dtype=torch.bfloat16) for _ in range(3))


@pytest.mark.parametrize("sink", [0, 3, np.int64(3), 3.0])
@pytest.mark.parametrize("kw", [
    dict(), dict(sliding_window=8.0), dict(sliding_window=np.int64(8)), dict(sliding_window=torch.tensor(8)),
    dict(scale=np.float32(0.5)), dict(scale=torch.tensor(0.5)), dict(scale=1), dict(softcap=np.float32(30)),
    dict(softcap=torch.tensor(30.0)), dict(softcap=30)])
def test_forward_and_backward(lib, kw, sink):
    kw = dict(dict(sliding_window=8), **kw, sink_tokens=sink)
    q, k, v = _qkv()
    attention.fastest_flash_attn_forward(q, k, v, causal=True, return_lse=True, **kw)
    assert lib.last[0] == ("ffa_fwd_sink" if sink else "ffa_fwd")
    assert lib.last[1][20] == 8
    attention.fastest_flash_attn_backward(q, q, k, v, q, torch.zeros(1, 2, 32), causal=True, **kw)
    assert lib.last[0] == ("ffa_bwd_sink" if sink else "ffa_bwd") and lib.last[1][28] == 8


@pytest.mark.parametrize("off", [5, np.int64(5), torch.tensor(5), 5.0])
@pytest.mark.parametrize("sink", [0, 3])
def test_offset(lib, off, sink):
    attention.flash_fwd(*_qkv(), scale=0.125, causal=True, q_offset=off, window=8, sink=sink)
    assert lib.last[1][19] == 5


def test_configuration_of_another_class(lib):
    """A configuration with the fields of the reference's, which has no sink_tokens."""
    from types import SimpleNamespace
    from fastest_flash_attention_b200 import AttentionConfig
    fields = {f: getattr(AttentionConfig(causal=True, sliding_window=8), f) for f in (
        "block_size_q", "block_size_kv", "causal", "sliding_window", "softcap", "num_kv_heads", "compute_dtype",
        "two_pass", "return_lse")}
    attention.fastest_flash_attn_forward(*_qkv(), config=SimpleNamespace(**fields))
    assert lib.last[0] == "ffa_fwd" and lib.last[1][18] == 1 and lib.last[1][20] == 8
    attention.fastest_flash_attn_forward(*_qkv(), config=SimpleNamespace(**fields), sink_tokens=2)
    assert lib.last[0] == "ffa_fwd_sink" and lib.last[1][21] == 2
    attention.fastest_flash_attn_forward(*_qkv(), config=AttentionConfig(**fields, sink_tokens=3), sink_tokens=2)
    assert lib.last[0] == "ffa_fwd_sink" and lib.last[1][21] == 3


def test_pools_of_one_page(lib):
    """A single page's stride says nothing about its size."""
    from fastest_flash_attention_b200 import copy_pages
    pool = torch.zeros(4096).as_strided((1, 2, 4, 8), (1 << 40, 32, 8, 1))
    assert pool.is_contiguous()
    copy_pages(pool, None, torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    import fastest_flash_attention_b200.kv_cache as kv
    ids = torch.zeros(1, dtype=torch.int32)
    original, kv._id_pair = kv._id_pair, lambda *a: (ids, ids)
    try:
        copy_pages(pool, None, ids, ids)
    finally:
        kv._id_pair = original
    assert lib.last[0] == "ffa_page_copy" and lib.last[1][6] == 2 * 4 * 8 * 4
