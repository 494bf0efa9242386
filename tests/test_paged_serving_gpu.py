"""The operators of a paged server together: page tables on the device, rotary
append, prefill of chunks, decoding behind a shared prefix, pages given back;
eager, and as one captured step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
H, HKV, D, PS = 8, 2, 64, 16


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _want(q, k, v, past):
    """64-bit causal attention: q [n, H, D] behind `past` of the tokens of k, v [t, HKV, D]."""
    kk, vv = (x.double().transpose(0, 1).repeat_interleave(H // HKV, 0) for x in (k, v))
    s = q.double().transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(D)
    hide = torch.arange(k.shape[0], device="cuda")[None, :] > past + torch.arange(q.shape[0], device="cuda")[:, None]
    return (torch.softmax(s.masked_fill(hide, -math.inf), -1) @ vv).transpose(0, 1)


def _close(o, want, v):
    # P and O rounded once each, and the fp32 terms (test_paged_prefill_gpu.py)
    return float((o.double() - want).abs().max()) <= float(v.abs().max()) * (2 * U[o.dtype] + 2.0 ** -10)


class _Server:
    """Six places of a batch over one pool; remembers every token's rotated key and value for the plain result."""

    def __init__(self, seed, dtype=torch.bfloat16):
        import fastest_flash_attention_b200 as ffa
        self.ffa = ffa
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.t = ffa.DevicePageTable(6, 64, 120, page_size=PS)
        self.kp, self.vp = (torch.full((120, HKV, PS, D), math.nan, device="cuda", dtype=dtype) for _ in range(2))
        self.cos, self.sin = ffa.rotary_tables(D, 2048, device="cuda")
        self.dtype = dtype
        self.k, self.v = ([torch.zeros(0, HKV, D, device="cuda", dtype=dtype) for _ in range(6)] for _ in range(2))

    def qkv(self, T):
        return [torch.randn(T, h, D, generator=self.g, device="cuda").to(self.dtype) for h in (H, HKV, HKV)]

    def append(self, new):
        T = sum(new)
        q, k, v = self.qkv(T)
        plan = self.t.assign(_ints(new), T)
        qr = self.ffa.rotary_append(q, k, v, self.cos, self.sin, plan.positions, plan.slots, self.kp, self.vp)
        kr = self.ffa.apply_rotary(k.transpose(0, 1)[None], None, self.cos, self.sin, plan.positions)[0][0].transpose(0, 1)
        at = 0
        for r, n in enumerate(new):
            self.k[r], self.v[r] = torch.cat([self.k[r], kr[at:at + n]]), torch.cat([self.v[r], v[at:at + n]])
            at += n
        return qr, plan

    def prefill(self, new):
        q, plan = self.append(new)
        o = self.ffa.paged_prefill(q, self.kp, self.vp, self.t.block_table, self.t.ctx_lens, plan.starts)
        at = 0
        for r, n in enumerate(new):
            if n:
                assert _close(o[at:at + n], _want(q[at:at + n], self.k[r], self.v[r], len(self.k[r]) - n), self.v[r]), r
            at += n

    def step(self, starts, prefixes):
        q, _ = self.append([1] * 6)
        o = self.ffa.prefix_decode(q, self.kp, self.vp, self.t.block_table, self.t.ctx_lens, _ints(starts),
                                   _ints(prefixes))
        for r in range(6):
            assert _close(o[r:r + 1], _want(q[r:r + 1], self.k[r], self.v[r], len(self.k[r]) - 1), self.v[r]), r


def test_serving_run():
    s = _Server(1)
    s.prefill([150, 33, 0, 0, 0, 0])      # a prompt with a system prompt of 144 tokens, another without
    s.t.share(0, [2, 3], 144)
    for r in (2, 3):
        s.k[r], s.v[r] = s.k[0][:144], s.v[0][:144]
    # rows 0, 2, 3 share: neighbours in the batch are rows 2 and 3, with row 0's pages
    s.prefill([0, 70, 5, 1, 20, 0])       # questions behind the prompt, a second chunk, a new request
    s.prefill([1, 1, 1, 1, 1, 60])
    for _ in range(3):
        s.step([2, 4], [144])
    s.t.release(torch.tensor([False, False, False, True, True, False], device="cuda"),
                keep=_ints([0, 0, 0, 144, 0, 0]))
    s.k[3], s.v[3] = s.k[3][:0], s.v[3][:0]
    s.k[4], s.v[4] = s.k[4][:0], s.v[4][:0]
    s.prefill([0, 0, 0, 40, 17, 0])       # other requests in their places, on the pages given back
    for _ in range(17):                   # over a page's end; groups of one
        s.step([0, 1, 2, 3], [16, 0, 33])
    s.t.release(torch.ones(6, dtype=torch.bool, device="cuda"), keep=_ints([0, 0, 144, 0, 0, 0]))
    assert s.t.num_free_pages == 120 and sorted(s.t.free_pages.tolist()) == list(range(120))


def test_captured_step_against_eager():
    """A step (tables, rotary append, decoding behind a prefix) in a graph, replayed across page boundaries: the same
    bits as eager steps."""
    a, b = _Server(2), _Server(2)
    for s in (a, b):
        s.prefill([100, 20, 0, 0, 31, 0])
        s.t.share(0, [2, 3], 96)
    starts, prefixes = _ints([2, 4]), _ints([96])
    ones = _ints([1] * 6)
    q, k, v = a.qkv(6)
    ffa = a.ffa

    def step(s):
        plan = s.t.assign(ones, 6)
        qr = ffa.rotary_append(q, k, v, s.cos, s.sin, plan.positions, plan.slots, s.kp, s.vp)
        return ffa.prefix_decode(qr, s.kp, s.vp, s.t.block_table, s.t.ctx_lens, starts, prefixes, max_prefix=96,
                                 max_own=512)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(_Server(3))
    torch.cuda.current_stream().wait_stream(st)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        out = step(a)
    for _ in range(40):
        for x, h in ((q, H), (k, HKV), (v, HKV)):
            x.copy_(torch.randn(6, h, D, generator=a.g, device="cuda"))
        want = step(b)
        gr.replay()
        assert torch.equal(out, want)
    assert torch.equal(a.t.block_table, b.t.block_table) and torch.equal(a.t.ctx_lens, b.t.ctx_lens)
    assert torch.equal(a.t.free_state, b.t.free_state)


def test_host_cache_prefill_and_shared_decode():
    from fastest_flash_attention_b200 import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(5)
    c = PagedKVCache(200, PS, HKV, D, torch.float16, "cuda")

    def rand(n, h):
        return torch.randn(n, h, D, generator=g, device="cuda").half()

    def append(s, n):
        c.append_tokens(s, *(rand(n, HKV).transpose(0, 1) for _ in range(2)))

    def plain(q, s, n):
        k, v = (x.transpose(0, 1) for x in c.get_kv(s))
        return _want(q, k, v, k.shape[0] - n), v
    append(0, 500)
    append(9, 77)
    c.fork_sequences([(0, 1), (0, 2)])
    c.fork_sequence(1, 3)
    new = {0: 3, 1: 40, 2: 1, 3: 17, 9: 5}
    for s, n in new.items():
        append(s, n)
    q = rand(sum(new.values()), H)
    o, lse = c.prefill(q, list(new), list(new.values()), return_lse=True)
    at = 0
    for s, n in new.items():
        want, v = plain(q[at:at + n], s, n)
        assert _close(o[at:at + n], want, v)
        at += n
    ids = [0, 1, 2, 3, 9]
    assert c.prefix_groups(ids) == ([0, 4, 5], [496, 0])
    q = rand(5, H)
    for softcap, ids in ((None, ids), (30.0, ids), (None, [1, 9, 2, 9, 3])):
        # (the last: neighbours that share nothing)
        o, lse = c.decode(q, ids, share_prefix=True, return_lse=True, softcap=softcap)
        o2, lse2 = c.decode(q, ids, return_lse=True, softcap=softcap)
        V = float(c.v_pages.abs().max())
        assert float((o.double() - o2.double()).abs().max()) <= 2 * V * (2 * U[torch.float16] + 2.0 ** -10)
        assert float((lse - lse2).abs().max()) <= 2 * 2.0 ** -10
