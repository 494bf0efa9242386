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


SIZES = [(1, 32, 1, 1024, 1024, 128, 128, 256, 4), (1, 4, 2, 100, 100, 64, 64, 16, 3), (2, 8, 8, 4096, 4096, 64, 64, 512, 300),
         (1, 2, 1, 640, 640, 192, 128, 65, 700), (1, 2, 2, 9000, 9000, 40, 24, 50, 5000), (1, 1, 1, 1, 1, 64, 64, 1, 1)]


@pytest.mark.parametrize("args", SIZES)
def test_each_type_alone(args):
    """What a type's kernels write and no more: the row statistics, and the
    fp32 sums of the shares, where queries are shared at all."""
    lib = _lib.load()
    B, Hq, Hkv, Sq, Skv, D, Dv, window, sinks = args
    plain = lib.ffa_bwd_workspace_size(B, Hq, Sq)
    width = 128 if max(D, Dv) <= 64 else 256 if D <= 128 else 320
    n_q, tiles = -(-Sq // 64), -(-min(sinks, Skv) // 128)
    parts = min(-(-n_q // (-(-(window + 128) // 64) + 1)), 64 // tiles if tiles <= 32 else 1)
    shares = B * Hkv * tiles * parts * 128 * width * 4 if parts > 1 else 0
    typed = {t: lib.ffa_bwd_sink_workspace_size_of(t, *args) for t in (0, 1, 2)}  # fp16, bf16, fp32
    assert typed[0] == typed[1] and plain + shares <= typed[0] <= plain + shares + 16
    assert typed[2] >= plain if (D, Dv) != (40, 24) else typed[2] == 0  # fp32 takes the exact widths
    assert lib.ffa_bwd_sink_workspace_size(*args) == max(typed.values())
    for bad in range(9):
        assert lib.ffa_bwd_sink_workspace_size_of(1, *args[:bad], 0, *args[bad + 1:]) == 0
    assert lib.ffa_bwd_sink_workspace_size_of(3, *args) == 0
