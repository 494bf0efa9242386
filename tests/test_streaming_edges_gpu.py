"""The streaming operators inside a CUDA graph, on a stream of their own, and on
pools whose offsets pass 32 bits.  Results are compared with the same calls in
the ordinary setting (bit for bit) or, for the long pools, with a copy of the
touched pages in a small pool."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(ffa, q, k, v, tables, pos, slots, kp, vp, bt, lens):
    """A decode step's two launches: rotate and append, then the windowed decode."""
    qr = ffa.rotary_append(q, k, v, *tables, pos, slots, kp, vp)
    return ffa.paged_decode(qr, kp, vp, bt, lens, sliding_window=100, sink_tokens=4, return_lse=True)


def _state(seed=0, R=5, Hq=8, Hkv=2, D=128, page=16, pages=100):
    import fastest_flash_attention_b200 as ffa
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    kp, vp = randn(pages, Hkv, page, D), randn(pages, Hkv, page, D)
    bt = torch.randperm(pages, generator=g, device="cuda")[:R * 15].view(R, 15).int()
    lens = torch.tensor([1, 30, 100, 180, 240], dtype=torch.int32, device="cuda")
    at = lens.long() - 1  # the new token is each context's last
    slots = (bt.gather(1, (at // page)[:, None])[:, 0] * page + at % page).int()
    return ffa, (randn(R, Hq, D), randn(R, Hkv, D), randn(R, Hkv, D), ffa.rotary_tables(D, 512), at.int(), slots, kp,
                 vp, bt, lens)


def test_decode_step_in_a_cuda_graph():
    ffa, st = _state()
    graph_st = [t.clone() if isinstance(t, torch.Tensor) else t for t in st]
    _step(ffa, *graph_st)  # warm-up outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(ffa, *graph_st)
    for seed in (1, 2):
        _, new = _state(seed)
        for dst, src in zip(graph_st, new):
            if isinstance(dst, torch.Tensor):
                dst.copy_(src)
        graph.replay()
        want = _step(ffa, *new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(graph_st[6], new[6]) and torch.equal(graph_st[7], new[7])


def test_on_a_stream_of_its_own():
    """Inputs made, operators called and results read on a side stream."""
    ffa, st = _state(3)
    want = _step(ffa, *st)
    x = torch.randn(1, 2, 300, 64, device="cuda")
    tables = ffa.rotary_tables(64, 512)

    def train(t):
        t = t.detach().requires_grad_()
        q, k = ffa.apply_rotary(t, t, *tables)
        o = ffa.fastest_flash_attn_func(q, k, t, causal=True, sliding_window=40, sink_tokens=3)
        return torch.autograd.grad(o, t, t.detach())[0]
    ref = train(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what follows is late unless it is on this stream too
        _, again = _state(3)
        got = _step(ffa, *again)
        g = train(x)
        ffa.copy_pages(again[6], again[7], again[8][0, :4], again[8][1, :4])
        ffa.move_tokens(again[6], again[7], again[8][2, :4] * 16, again[8][3, :4] * 16)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(g, ref)
    for pool, src in ((again[6], st[6]), (again[7], st[7])):
        assert torch.equal(pool[again[8][1, :4].long()], src[st[8][0, :4].long()])
        assert torch.equal(pool[again[8][3, :4].long(), :, 0], src[st[8][2, :4].long(), :, 0])


def test_pools_past_32_bit_offsets():
    """2.3e9 values a pool: the last pages' offsets pass 2^31 elements and 2^32 bytes."""
    import fastest_flash_attention_b200 as ffa
    P, Hkv, page, D = 70000, 8, 32, 128
    kp, vp = (torch.zeros(P, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    ids = torch.tensor([P - 1, 65536, P - 7, 3], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    small_k, small_v = (torch.randn(4, Hkv, page, D, generator=g, device="cuda").half() for _ in range(2))
    kp[ids], vp[ids] = small_k, small_v
    q, k, v = (torch.randn(1, h, D, generator=g, device="cuda").half() for h in (16, Hkv, Hkv))
    lens = torch.tensor([4 * page], dtype=torch.int32, device="cuda")
    tables = ffa.rotary_tables(D, 256)
    pos = torch.tensor([4 * page - 1], device="cuda")
    outs = []
    for kk, vv, bt in ((kp, vp, ids), (small_k, small_v, torch.arange(4, device="cuda"))):
        slot = (bt[3:] * page + page - 1).int()
        qr = ffa.rotary_append(q, k, v, *tables, pos, slot, kk, vv)
        outs.append(ffa.paged_decode(qr, kk, vv, bt[None].int(), lens, sliding_window=90, sink_tokens=20))
    assert torch.equal(*outs)
    assert torch.equal(kp[ids], small_k) and torch.equal(vp[ids], small_v)
    ffa.copy_pages(kp, vp, [P - 1, 65536], [P - 2, 69000])
    ffa.move_tokens(kp, vp, [(P - 7) * page + 5], [(P - 3) * page + 31])
    assert torch.equal(kp[P - 2], small_k[0]) and torch.equal(vp[69000], small_v[1])
    assert torch.equal(kp[P - 3, :, 31], small_k[2, :, 5]) and not bool(kp[P - 3, :, :31].any())
