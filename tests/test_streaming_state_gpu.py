"""The streaming operators at arguments of unusual type, layout or size on the
GPU: the same results, bit for bit, as the ordinary form of the same call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pools(P=8, Hkv=2, page=16, D=64, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(P, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))


def _reports(call):
    """Whether the call's bad ids were reported (tests read the error word after every call)."""
    with pytest.raises(RuntimeError, match="FFA_ERR_INVALID_ARG"):
        call()


@pytest.mark.parametrize("bad", [2 ** 32 + 5, 2 ** 33, -2 ** 32 + 5, 2 ** 31, 2 ** 62])
def test_64_bit_ids_do_not_wrap(bad):
    """An id outside 32 bits must not turn into one inside the pool."""
    import fastest_flash_attention_b200 as ffa
    k, v = _pools()
    k0, v0 = k.clone(), v.clone()
    for fn in (ffa.copy_pages, ffa.move_tokens):
        for src, dst in (([bad, 1], [2, 3]), ([1, 2], [3, bad])):
            _reports(lambda: fn(k, v, torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")))
    # only what the good ids name has changed: page 2 or 3 (pages), token 2 or 3 of page 0 (tokens)
    for now, then in ((k, k0), (v, v0)):
        assert torch.equal(now[4:], then[4:]) and torch.equal(now[1], then[1]) and torch.equal(now[0, :, 4:], then[0, :, 4:])
    q = torch.randn(1, 4, 64, device="cuda").to(torch.bfloat16)
    bt, lens = torch.tensor([[1, 2]], device="cuda"), torch.tensor([20], device="cuda")
    want = ffa.paged_decode(q, k, v, bt.int(), lens.int(), sliding_window=8, sink_tokens=2)
    assert torch.equal(ffa.paged_decode(q, k, v, bt, lens, sliding_window=8, sink_tokens=2), want)
    _reports(lambda: ffa.paged_decode(q, k, v, torch.tensor([[1, bad]], device="cuda"), lens, sliding_window=8))
    _reports(lambda: ffa.paged_decode(q, k, v, bt, torch.tensor([bad], device="cuda"), sliding_window=8))


@pytest.mark.parametrize("form", ["odd strides", "odd base"])
def test_decode_of_queries_that_only_look_contiguous(form):
    """A tensor of one row counts as contiguous whatever its outer strides are, and at any address."""
    import fastest_flash_attention_b200 as ffa
    k, v = _pools(Hkv=1)
    bt = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    src = torch.randn(1, 1, 64, device="cuda").to(torch.bfloat16)
    if form == "odd strides":
        q = torch.empty(200, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 64), (67, 65, 1)).copy_(src)
    else:
        q = torch.empty(65, dtype=torch.bfloat16, device="cuda")[1:].view(1, 1, 64).copy_(src)
    assert q.is_contiguous()
    want = ffa.paged_decode(src, k, v, bt, lens, sliding_window=8, sink_tokens=2)
    assert torch.equal(ffa.paged_decode(q, k, v, bt, lens, sliding_window=8, sink_tokens=2), want)


@pytest.mark.parametrize("form", ["odd strides", "zero strides", "odd base"])
def test_attention_of_operands_that_only_look_contiguous(form):
    from fastest_flash_attention_b200 import fastest_flash_attn_func
    g = torch.Generator(device="cuda").manual_seed(1)
    src = [torch.randn(1, 1, 40, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(4)]

    def odd(t):
        if form == "odd strides":
            return torch.empty(4000, dtype=t.dtype, device="cuda").as_strided(t.shape, (2601, 2567, 64, 1)).copy_(t)
        if form == "zero strides":
            return torch.empty(4000, dtype=t.dtype, device="cuda").as_strided(t.shape, (0, 0, 64, 1)).copy_(t)
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    def run(q, k, v, do, **kw):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = fastest_flash_attn_func(q, k, v, causal=True, sliding_window=16, **kw)
        return (o,) + torch.autograd.grad(o, (q, k, v), do)
    for kw in (dict(sink_tokens=3), dict()):
        for a, b in zip(run(*map(odd, src), **kw), run(*src, **kw)):
            assert torch.equal(a, b)


def _sink_call(lib, _lib, q, k, v, window, sinks, do=None, skv=None):
    """ffa_fwd_sink (and, with do, ffa_bwd_sink) through the C entry points."""
    B, Hq, Sq, D = q.shape
    Hkv, Skv, Dv = k.shape[1], k.shape[2] if skv is None else skv, v.shape[3]
    o = torch.empty(B, Hq, Sq, Dv, dtype=q.dtype, device="cuda")
    lse = torch.empty(B, Hq, Sq, device="cuda")
    st = [_lib.strides3(t) for t in (q, k, v, o)]
    stream = _lib.stream_of(q)
    sizes = (_lib.DTYPE_CODE[q.dtype], B, Hq, Hkv, Sq, Skv, D, Dv)
    _lib.check(lib.ffa_fwd_sink(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), *sizes, *st,
                                0.125, 1, 0, window, sinks, 0.0, None, stream), "ffa_fwd_sink")
    if do is None:
        return o, lse
    grads = [torch.empty_like(t) for t in (q, k, v)]
    ws = torch.empty(lib.ffa_bwd_sink_workspace_size(B, Hq, Hkv, Sq, Skv, D, Dv, window, sinks), dtype=torch.uint8,
                     device="cuda")
    _lib.check(lib.ffa_bwd_sink(
        do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
        *(t.data_ptr() for t in grads), *sizes, *st, _lib.strides3(do), *map(_lib.strides3, grads), 0.125, 1, 0, window,
        sinks, 0.0, ws.data_ptr(), ws.numel(), None, stream), "ffa_bwd_sink")
    return (o, lse, *grads)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30 + 1])
def test_c_entry_points_with_windows_near_2_31(window):
    """A window past every length hides nothing: the same as one of 2^20."""
    from fastest_flash_attention_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, do = (torch.randn(1, 2, 300, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(4))
    lib = _lib.load()
    want = _sink_call(lib, _lib, q, k, v, 2 ** 20, 4, do)
    assert bool(want[3][0, :, 4:].any(-1).all())  # every key has a gradient
    for a, b in zip(_sink_call(lib, _lib, q, k, v, window, 4, do), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,Dv", [(64, 64), (40, 24), (136, 72)])
def test_c_forward_of_no_keys(D, Dv):
    """No key: 0 and -inf, at every head dim that the entry point takes."""
    from fastest_flash_attention_b200 import _lib
    q, k, v = (torch.randn(1, 2, 8, d, device="cuda").to(torch.bfloat16) for d in (D, D, Dv))
    o, lse = _sink_call(_lib.load(), _lib, q, k, v, 4, 2, skv=0)
    assert not bool(o.any()) and bool((lse == -float("inf")).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,Dv,window,sinks", [
    (1, 8, 1, 1024, 128, 128, 256, 4), (1, 4, 2, 216, 64, 64, 48, 4), (2, 2, 2, 1300, 64, 64, 100, 300),
    (1, 2, 1, 640, 192, 128, 65, 700), (1, 2, 2, 5000, 64, 64, 50, 4500)])
def test_backward_stays_inside_its_workspace(B, Hq, Hkv, S, D, Dv, window, sinks, dtype):
    """Nothing past the bytes that the size function of the type names is written."""
    from fastest_flash_attention_b200 import _lib, attention
    lib = _lib.load()
    g = torch.Generator(device="cuda").manual_seed(S)
    q, k, v, do = (torch.randn(B, h, S, d, generator=g, device="cuda").to(dtype)
                   for h, d in ((Hq, D), (Hkv, D), (Hkv, Dv), (Hq, Dv)))
    o, lse = attention.flash_fwd(q, k, v, scale=0.125, causal=True, window=window, sink=sinks)
    want = attention.flash_bwd(do, q, k, v, o, lse, scale=0.125, causal=True, window=window, sink=sinks)
    sizes = (attention._ATTN_DTYPE_CODE[dtype], B, Hq, Hkv, S, S, D, Dv)
    size = lib.ffa_bwd_sink_workspace_size_of(*sizes, window, sinks)
    ws = torch.full((size + 1024,), 0xAB, dtype=torch.uint8, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    ts = (q, k, v, o, do, *grads)
    _lib.check(lib.ffa_bwd_sink(do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                                *(t.data_ptr() for t in grads), *sizes, *map(_lib.strides3, ts), 0.125, 1, 0, window,
                                sinks, 0.0, ws.data_ptr(), size, None, _lib.stream_of(q)), "ffa_bwd_sink")
    assert bool((ws[size:] == 0xAB).all()) and all(torch.equal(a, b) for a, b in zip(grads, want))
    assert lib.ffa_bwd_sink(do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                            *(t.data_ptr() for t in grads), *sizes, *map(_lib.strides3, ts), 0.125, 1, 0, window,
                            sinks, 0.0, ws.data_ptr(), size - 1, None, _lib.stream_of(q)) == _lib.FFA_ERR_WORKSPACE
