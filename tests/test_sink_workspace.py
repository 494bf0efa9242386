"""The workspace of the backward with sinks: what its size function answers is
what the call wants (no kernel is launched, so no GPU is needed)."""
import pytest

from fastest_flash_attention_b200 import _lib


def _call(lib, size, B, Hq, Hkv, Sq, Skv, D, Dv, window, sinks):
    s, p = _lib.i64arr(64, 64, 64), 4096  # never dereferenced: the call ends before a launch
    return lib.ffa_bwd_sink(p, p, p, p, p, p, p, p, p, 1, B, Hq, Hkv, Sq, Skv, D, Dv, s, s, s, s, s, s, s, s, 1.0, 1, 0,
                            window, sinks, 0.0, p, size, None, None)


def test_no_sinks():
    """No size is given for a call without sinks (ffa_bwd's), so the call is refused for that, not for its workspace."""
    lib = _lib.load()
    args = (1, 4, 2, 100, 100, 64, 64, 16, 0)
    size = lib.ffa_bwd_sink_workspace_size(*args)
    assert size == 0 and _call(lib, size, *args) == _lib.FFA_ERR_INVALID_ARG
    assert "ffa_bwd" in lib.ffa_last_error().decode()
