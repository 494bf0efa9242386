"""Host side of the long-context streaming operators: rotary tables against
their formulas in 64 bits, refusals, and the page bookkeeping of forks, trims
and compactions on a host-side pool."""
import math

import pytest
import torch

import fastest_flash_attention_b200 as ffa


def test_rotary_tables_plain_and_linear():
    cos, sin = ffa.rotary_tables(8, 100000, 10000.0, device="cpu")
    assert cos.shape == (100000, 4) and cos.dtype == torch.float32
    for p, i in ((0, 0), (1, 3), (99999, 0), (54321, 1)):
        a = p * 10000.0 ** (-2 * i / 8)
        # fp32 rounding of a value below 1, and the 64-bit angle's own rounding
        assert abs(float(cos[p, i]) - math.cos(a)) <= 2.0 ** -24 and abs(float(sin[p, i]) - math.sin(a)) <= 2.0 ** -24
    half, _ = ffa.rotary_tables(8, 10, 10000.0, scaling="linear", factor=2.0, device="cpu")
    full, _ = ffa.rotary_tables(8, 10, 10000.0, device="cpu")
    assert torch.equal(half[::2], full[:5])


def test_rotary_tables_ntk_and_yarn():
    def angles(**kw):
        cos, sin = ffa.rotary_tables(64, 2, 10000.0, device="cpu", **kw)
        return torch.atan2(sin[1].double(), cos[1].double()), float((cos[1] ** 2 + sin[1] ** 2).sqrt().mean())
    plain, _ = angles()
    ntk, m = angles(scaling="ntk", factor=8.0)
    # 2^-22: two fp32 table entries behind an angle of at most 1
    assert abs(float(ntk[0] - plain[0])) <= 2.0 ** -22 and abs(float(ntk[-1] * 8 / plain[-1]) - 1) <= 1e-6
    assert abs(m - 1) <= 1e-6
    yarn, m = angles(scaling="yarn", factor=8.0, original_max_len=4096)
    assert abs(float(yarn[0] - plain[0])) <= 2.0 ** -22 and abs(float(yarn[-1] * 8 / plain[-1]) - 1) <= 1e-6
    assert abs(m - (0.1 * math.log(8.0) + 1)) <= 1e-6
    ratio = yarn / plain
    assert bool((ratio[1:] <= ratio[:-1] + 1e-6).all())  # from the plain frequencies down to the divided ones


@pytest.mark.parametrize("kw", [
    dict(dim=7, max_len=4), dict(dim=0, max_len=4), dict(dim=8, max_len=0), dict(dim=8, max_len=4, factor=0.0),
    dict(dim=8, max_len=4, scaling="yarn", factor=2.0), dict(dim=8, max_len=4, scaling="cubic"),
    dict(dim=2, max_len=4, scaling="ntk", factor=2.0),
])
def test_rotary_tables_refusals(kw):
    with pytest.raises(ValueError):
        ffa.rotary_tables(device="cpu", **kw)


def test_c_entry_points_refuse_sizes_that_mean_nothing():
    """No size crashes an entry point: it returns a status (no kernel is launched, so no GPU is needed)."""
    from fastest_flash_attention_b200 import _lib
    lib = _lib.load()
    good = dict(B=1, Hq=4, Hkv=2, Sq=8, Skv=8, D=64, Dv=64, window=4, sinks=2)
    assert lib.ffa_bwd_sink_workspace_size(*good.values()) > 0
    for name in ("B", "Hq", "Hkv", "Sq", "Skv", "window", "sinks"):
        for bad in (0, -1, -2 ** 31):
            assert lib.ffa_bwd_sink_workspace_size(*dict(good, **{name: bad}).values()) == 0
    s, p = _lib.i64arr(64, 64, 64), 4096  # never dereferenced: the sizes are refused first
    for B, Hq, Hkv, Sq, Skv, D, Dv, w, n in ((0, 4, 2, 8, 8, 64, 64, 4, 2), (1, 4, 0, 8, 8, 64, 64, 4, 2),
                                             (1, 3, 2, 8, 8, 64, 64, 4, 2), (1, 4, 2, -1, 8, 64, 64, 4, 2),
                                             (1, 4, 2, 8, 8, 65, 64, 4, 2), (1, 4, 2, 8, 8, 64, 136, 4, 2),
                                             (1, 4, 2, 8, 8, 64, 64, 0, 2), (1, 4, 2, 8, 8, 64, 64, 4, -1)):
        assert lib.ffa_fwd_sink(p, p, p, p, p, 1, B, Hq, Hkv, Sq, Skv, D, Dv, s, s, s, s, 1.0, 1, 0, w, n, 0.0, None,
                                None) in (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
        assert lib.ffa_bwd_sink(p, p, p, p, p, p, p, p, p, 1, B, Hq, Hkv, Sq, Skv, D, Dv, s, s, s, s, s, s, s, s, 1.0,
                                1, 0, w, n, 0.0, p, 1 << 30, None,
                                None) in (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
    for R, Hq, Hkv, D, P, page, width, w, n in ((-1, 4, 2, 64, 4, 16, 2, 4, 0), (1, 4, 0, 64, 4, 16, 2, 4, 0),
                                                (1, 5, 2, 64, 4, 16, 2, 4, 0), (1, 4, 2, 60, 4, 16, 2, 4, 0),
                                                (1, 4, 2, 136, 4, 16, 2, 4, 0), (1, 4, 2, 64, 0, 16, 2, 4, 0),
                                                (1, 4, 2, 64, 4, 0, 2, 4, 0), (1, 4, 2, 64, 4, 16, 0, 4, 0),
                                                (1, 4, 2, 64, 4, 16, 2, 0, 0), (1, 4, 2, 64, 4, 16, 2, 4, -1),
                                                (1, 4, 2, 64, 2 ** 30, 2 ** 20, 2, 4, 0)):
        assert lib.ffa_window_decode(p, p, p, p, p, p, None, 1, R, Hq, Hkv, D, P, page, width, s, s, 1.0, 0.0, w, n, 0,
                                     None, None) in (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
    assert lib.ffa_page_copy(p, None, p, p, -1, 4, 32, None, None) == _lib.FFA_ERR_INVALID_ARG
    assert lib.ffa_page_copy(p, None, p, p, 1, 4, 33, None, None) == _lib.FFA_ERR_UNSUPPORTED
    assert lib.ffa_token_move(p, None, p, p, 1, 2, 0, 4, 32, None, None) == _lib.FFA_ERR_INVALID_ARG
    assert lib.ffa_rotary(p, s, p, s, None, None, None, None, p, p, 8, p, 0, 0, 1, 1, 1, 4, 0, 64, 63, 0, 0, None,
                          None) == _lib.FFA_ERR_INVALID_ARG
    assert lib.ffa_rotary(p, s, p, s, p, None, p, s, p, p, 8, p, 0, 0, 1, 1, 1, 4, 2, 64, 64, 0, 0, None,
                          None) == _lib.FFA_ERR_INVALID_ARG
    assert lib.ffa_rotary_append(p, s, p, s, p, s, p, s, p, p, 0, p, 0, p, p, p, 1, 1, 4, 2, 64, 64, 0, 16, 4, None,
                                 None) == _lib.FFA_ERR_INVALID_ARG


def test_direct_calls_check_their_arguments():
    """The module that calls the library without ctypes raises for what does not fit a parameter."""
    from fastest_flash_attention_b200 import _lib
    call = _lib.direct()
    assert set(call.NAMES) <= set(_lib.SIGNATURES)
    ok = (0, None, 0, 0, 0, 4, 32, None, None)  # n = 0: nothing to do
    assert call.ffa_page_copy(*ok) == _lib.FFA_OK
    with pytest.raises(TypeError):
        call.ffa_page_copy(*ok[:-1])
    with pytest.raises(TypeError):
        call.ffa_page_copy(0, None, 0, 0, 0.5, 4, 32, None, None)
    with pytest.raises(OverflowError):
        call.ffa_page_copy(0, None, 0, 0, 0, 2 ** 31, 32, None, None)
    with pytest.raises(KeyError):
        call.bind("ffa_nothing", 0)
    args = [4096] * 7 + [1, -1, 4, 2, 64, 4, 16, 2, (1, 1), (1, 1), 1.0, 0, 4, 0, 0, None, None]
    assert call.ffa_window_decode(*args) == _lib.FFA_ERR_INVALID_ARG
    for i, bad, err in ((15, [1, 1], TypeError), (15, (1,) * 5, TypeError), (16, (1, "a"), TypeError),
                        (17, "x", TypeError), (0, 1.5, TypeError), (7, 2 ** 40, OverflowError)):
        with pytest.raises(err):
            call.ffa_window_decode(*args[:i], bad, *args[i + 1:])


def test_new_operators_refuse_cpu_tensors():
    x = torch.zeros(1, 1, 2, 8)
    cos, sin = ffa.rotary_tables(8, 4, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.apply_rotary(x, None, cos, sin)
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.copy_pages(x, None, [0], [0])
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.move_tokens(x, None, [0], [0])


def _cache(pages=32, ps=4):
    return ffa.PagedKVCache(max_pages=pages, page_size=ps, num_heads=2, head_dim=4, dtype=torch.float32)


def _tokens(n, base=0):
    k = (torch.arange(n, dtype=torch.float32) + base)[None, :, None].expand(2, n, 4).contiguous()
    return k, -k


def test_fork_shares_full_pages_and_copies_the_last():
    c = _cache()
    c.append_tokens("a", *_tokens(10))
    c.fork_sequence("a", "b")
    ta, tb = c.sequences["a"]["page_table"], c.sequences["b"]["page_table"]
    assert ta[:2] == tb[:2] and ta[2] != tb[2] and c.num_free_pages == 32 - 4
    c.append_tokens("b", *_tokens(3, 100))
    assert c.get_kv("a")[0][0, :, 0].tolist() == list(range(10))
    assert c.get_kv("b")[0][0, :, 0].tolist() == list(range(10)) + [100, 101, 102]
    c.free_sequence("a")
    assert c.num_free_pages == 32 - 4  # a's own last page back, b's new one gone
    c.free_sequence("b")
    assert sorted(c.free_pages) == list(range(32)) and not c._more_owners


def test_fork_on_a_page_boundary_and_empty():
    c = _cache()
    c.append_tokens(0, *_tokens(8))
    c.append_tokens(5, *_tokens(0))
    c.fork_sequences([(0, 1), (5, 6)])
    assert c.num_free_pages == 30 and c.sequences[6]["len"] == 0
    c.append_tokens(1, *_tokens(1, 50))
    assert c.get_kv(1)[0][0, :, 0].tolist() == list(range(8)) + [50] and c.get_kv(0)[0].shape[1] == 8


def test_fork_refusals_change_nothing():
    c = _cache(pages=3)
    c.append_tokens(0, *_tokens(9))
    for pairs, err in (([(1, 2)], KeyError), ([(0, 0)], ValueError), ([(0, 2), (0, 2)], ValueError),
                       ([(0, 2)], RuntimeError)):
        with pytest.raises(err):
            c.fork_sequences(pairs)
        assert list(c.sequences) == [0] and c.num_free_pages == 0 and not c._more_owners


def test_trim_frees_pages_outside_window_and_sinks():
    c = _cache()
    c.append_tokens(0, *_tokens(30))
    assert c.trim_sequence(0, 9, 5) == 3  # tokens 8..19 in pages 2, 3, 4; 21 is the window's first
    assert [p < 0 for p in c.sequences[0]["page_table"]] == [False] * 2 + [True] * 3 + [False] * 3
    assert c.trim_sequence(0, 9, 5) == 0
    bt, lens = c.block_table([0], sliding_window=9, sink_tokens=5)
    assert lens.tolist() == [30] and bt.shape == (1, 8)
    with pytest.raises(ValueError):  # the whole context is no longer there
        c.block_table([0])
    with pytest.raises(RuntimeError):
        c.get_kv(0)
    c.append_tokens(0, *_tokens(7, 30))
    assert c.sequences[0]["len"] == 37
    c.free_sequence(0)
    assert sorted(c.free_pages) == list(range(32))


def test_compact_keeps_window_and_sinks():
    c = _cache()
    c.append_tokens(0, *_tokens(30))
    c.append_tokens(1, *_tokens(6))
    c.trim_sequence(0, 9, 5)
    assert c.compact_sequences([0, 1], 9, 5) == 16  # sequence 1 fits and stays as it is
    assert c.get_kv(0)[0][0, :, 0].tolist() == list(range(5)) + list(range(21, 30))
    assert c.get_kv(1)[1].shape[1] == 6
    assert c.position(0) == 30 and c.position(1) == 6 and c.position("none") == 0
    assert c.num_free_pages == 32 - 4 - 2
    assert c.compact_sequences([0], 9, 5) == 0


def test_compact_refusals_change_nothing():
    c = _cache(pages=8)
    c.append_tokens(0, *_tokens(32))
    table = list(c.sequences[0]["page_table"])
    with pytest.raises(RuntimeError):  # no page left to move to
        c.compact_sequences([0], 9, 5)
    with pytest.raises(KeyError):
        c.compact_sequences([3], 9)
    with pytest.raises(ValueError):
        c.compact_sequences([0, 0], 9)
    for w, n in ((0, 0), (-3, 0), (4, -1)):
        with pytest.raises(ValueError):
            c.compact_sequences([0], w, n)
        with pytest.raises(ValueError):
            c.trim_sequence(0, w, n)
    c.trim_sequence(0, 9, 5)
    assert c.num_free_pages == 3  # tokens 8..19
    with pytest.raises(RuntimeError, match="freed"):  # a wider window than what is left
        c.compact_sequences([0], 13, 0)  # from token 19 on
    assert c.sequences[0]["len"] == 32 and c.sequences[0]["page_table"][:2] == table[:2] and c.num_free_pages == 3
