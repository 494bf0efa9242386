"""Several new tokens of each request against its pages, against a plain 64-bit
attention of each request.

Tolerances, derived beforehand.  u = half a step of the data's type relative to a
value (2^-8 bf16, 2^-11 fp16).  P is rounded to it (its rounding moves O by at
most u V, V the largest value) and O is rounded once more: 2 u V.  The fp32
terms: a score of magnitude S <= 40 carries at most (D + 8) 2^-24 S <= 2^-11.6
for D <= 128, which moves the LSE by as much and O by 2 V times as much; fp16 P
below 2^-14 has an absolute error of 2^-25, over at most 2^13 keys 2^-12 V;
2^x and lg2 are good to 2^-21.  So |O error| <= V (2 u + 2^-10), |LSE error| <=
2^-10."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lens, page, Hkv, D, dtype, seed, garbage=True):
    """Pools and a permuted block table; what no request reads is NaN, -1 in the table."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    P = sum(pages) + 2
    kp, vp = (torch.full((P, Hkv, page, D), math.nan, device="cuda", dtype=dtype) for _ in range(2))
    ids = torch.randperm(P, generator=g, device="cuda").tolist()
    bt = torch.full((len(lens), max(1, max(pages))), -1 if garbage else 0, dtype=torch.int32)
    for r, n in enumerate(lens):
        for i in range(pages[r]):
            bt[r, i] = ids.pop()
        if n:
            tok = torch.arange(n, device="cuda")
            pg = bt[r].cuda()[tok // page].long()
            for pool in (kp, vp):
                pool[pg, :, tok % page] = torch.randn(n, Hkv, D, generator=g, device="cuda").to(dtype)
    return kp, vp, bt.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), g


def want_of(q, kp, vp, bt, row, n, past, softcap=None, scale=None):
    """64-bit attention of q [m, Hq, D] over a row's first n tokens; query i sees the first past + i + 1."""
    m, Hq, D = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    tok = torch.arange(n, device="cuda")
    pg = bt[row].long()[tok // page]
    k, v = (x[pg, :, tok % page].double().transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for x in (kp, vp))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) * (scale or 1 / math.sqrt(D))
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.masked_fill(tok[None, :] > past + torch.arange(m, device="cuda")[:, None], -math.inf)
    return (torch.softmax(s, -1) @ v).transpose(0, 1), torch.logsumexp(s, -1).transpose(0, 1), float(v.abs().max())


def check(q, kp, vp, bt, lens, new, o, lse, softcap=None, scale=None):
    at = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        if m:
            want, wl, V = want_of(q[at:at + m], kp, vp, bt, r, n, n - m, softcap, scale)
            assert float((o[at:at + m].double() - want).abs().max()) <= V * (2 * U[q.dtype] + 2.0 ** -10), r
            if lse is not None:
                assert float((lse[at:at + m].double() - wl).abs().max()) <= 2.0 ** -10, r
        at += m


def starts_of(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


CASES = [
    # lens, new, page, Hq, Hkv, D, softcap, dtype
    ([1], [1], 16, 1, 1, 64, None, torch.bfloat16),                          # one token
    ([5, 0, 16, 17, 300], [5, 0, 1, 17, 2], 16, 8, 2, 64, None, torch.float16),  # an empty request, page edges
    ([127, 128, 129, 255, 257], [127, 128, 129, 1, 129], 8, 4, 4, 128, None, torch.bfloat16),  # tile edges, tiny pages
    ([1000, 70], [900, 70], 24, 21, 3, 96, 30.0, torch.float16),             # seven heads a group, head dim 96, softcap
    ([2500], [3], 64, 32, 8, 128, None, torch.bfloat16),                     # few rows: the context is split
    ([5000, 3, 4000], [1, 2, 300], 128, 8, 1, 128, None, torch.float16),     # one kv head, split, uneven
    ([700, 333], [64, 333], 256, 34, 1, 72, 2.0, torch.bfloat16),            # group of 34, a tight cap, big pages
    ([400, 20], [9, 20], 40, 128, 1, 8, None, torch.float16),                # group of 128, head dim 8, page 40
    ([33] * 70, [1] * 70, 16, 16, 8, 128, 50.0, torch.bfloat16),             # more requests than a warp's lanes
    ([6000], [1500], 16, 4, 1, 64, None, torch.bfloat16),
    # more requests than lanes, of no token, one block and several
    ([(37 * i) % 300 + i % 3 for i in range(45)], [((37 * i) % 300 + i % 3) // (1 + i % 4) for i in range(45)], 16, 12, 3,
     64, None, torch.float16),
    ([900 + i for i in range(40)], [(i * 29) % 90 for i in range(40)], 64, 8, 2, 128, None, torch.bfloat16),
]


@pytest.mark.parametrize("lens,new,page,Hq,Hkv,D,softcap,dtype", CASES)
def test_prefill(lens, new, page, Hq, Hkv, D, softcap, dtype):
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, ln, g = make(lens, page, Hkv, D, dtype, len(lens) + D)
    T = sum(new)
    q = torch.randn(T, Hq, D, generator=g, device="cuda").to(dtype)
    st = starts_of(new)
    o, lse = paged_prefill(q, kp, vp, bt, ln, st, softcap=softcap, return_lse=True)
    check(q, kp, vp, bt, lens, new, o, lse, softcap)
    # strided heads, another scale, hints that split differently, tokens behind the last request, given output
    wide = torch.full((T + 3, Hq, D + 8), math.nan, device="cuda", dtype=dtype)
    wide[:T, :, :D] = q
    for max_ctx in (1, max(lens), 50 * max(lens)):
        out = torch.full((T + 3, Hq, D), 7.0, device="cuda", dtype=dtype)
        o2 = paged_prefill(wide[..., :D], kp, vp, bt.long(), ln.long(), st.long(), softcap=softcap, scale=0.3,
                           max_ctx=max_ctx, out=out)
        assert o2 is out and bool((out[T:] == 7).all())
        check(q, kp, vp, bt, lens, new, o2, None, softcap, 0.3)


def test_two_runs_give_the_same_bits():
    from fastest_flash_attention_b200 import paged_prefill
    lens, new = [3000, 800, 41], [5, 200, 41]
    kp, vp, bt, ln, g = make(lens, 32, 2, 128, torch.bfloat16, 1)
    q = torch.randn(sum(new), 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    a = paged_prefill(q, kp, vp, bt, ln, starts_of(new), return_lse=True)
    b = paged_prefill(q, kp, vp, bt, ln, starts_of(new), return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_scores_and_infinite_ones():
    """Scores far apart (the maximum moves by more than the lazy rescale allows), and a key of infinities that
    only later queries see."""
    from fastest_flash_attention_b200 import paged_prefill
    n = 400
    kp, vp, bt, ln, g = make([n], 16, 1, 64, torch.float16, 9)
    order = bt[0].long()
    ramp = torch.linspace(-12, 12, n, device="cuda")  # scores rise along the context: every tile rescales
    tok = torch.arange(n, device="cuda")
    kp[order[tok // 16], 0, tok % 16] = (ramp[:, None] * torch.ones(64, device="cuda") / 8).half()
    q = torch.full((n, 1, 64), 4.0, device="cuda", dtype=torch.float16)
    o, lse = paged_prefill(q, kp, vp, bt, ln, starts_of([n]), return_lse=True)
    check(q, kp, vp, bt, [n], [n], o, lse)
    kp[order[300 // 16], 0, 300 % 16] = -math.inf  # q > 0: a score of -inf, as a mask of the caller's
    o2, lse2 = paged_prefill(q, kp, vp, bt, ln, starts_of([n]), return_lse=True)
    assert torch.equal(o2[:300], o[:300]) and torch.equal(lse2[:300], lse[:300])
    keep = tok != 300
    for i in (300, 301, 399):
        s = (kp[order[tok // 16], 0, tok % 16].double() @ q[i, 0].double() / 8)[:i + 1][keep[:i + 1]]
        v = vp[order[tok // 16], 0, tok % 16].double()[:i + 1][keep[:i + 1]]
        assert float((o2[i, 0].double() - torch.softmax(s, -1) @ v).abs().max()) <= float(v.abs().max()) * (
            2 * U[torch.float16] + 2.0 ** -10)


def test_data_that_means_nothing_is_reported():
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, ln, g = make([40, 30], 16, 2, 64, torch.float16, 3, garbage=False)
    q = torch.randn(12, 4, 64, generator=g, device="cuda").to(torch.float16)
    st = starts_of([8, 4])

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    for kw, word in ((dict(st=ints(0, 8, 13)), "boundaries"), (dict(st=ints(0, 8, 7)), "boundaries"),
                     (dict(st=ints(-1, 8, 12)), "boundaries"), (dict(ln=ints(40, 3)), "context length"),
                     (dict(ln=ints(7, 30)), "context length"), (dict(ln=ints(40, -1)), "context length"),
                     (dict(ln=ints(40, 1000)), "context length"), (dict(bt=bt * 0 + 99), "block-table entry"),
                     (dict(bt=bt * 0 - 1), "block-table entry"), (dict(bt=bt.long() + 2 ** 32), "block-table entry"),
                     (dict(st=st.long() + 2 ** 32), "boundaries"), (dict(ln=ln.long() + 2 ** 32), "context length")):
        a = dict(dict(bt=bt, ln=ln, st=st), **kw)
        with pytest.raises(RuntimeError, match=word):
            paged_prefill(q, kp, vp, a["bt"], a["ln"], a["st"])
    o = paged_prefill(q, kp, vp, bt, ln, st)
    check(q, kp, vp, bt, [40, 30], [8, 4], o, None)


def test_captured_and_replayed_on_a_side_stream():
    """Two graphs of one call (their workspaces are their own), replayed with other contents, on a stream of
    their own; eager calls between."""
    from fastest_flash_attention_b200 import paged_prefill
    lens, new = [2000, 900], [2, 3]
    kp, vp, bt, ln, g = make(lens, 16, 2, 128, torch.bfloat16, 4)
    q = torch.randn(5, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    st = starts_of(new)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged_prefill(q, kp, vp, bt, ln, st)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = paged_prefill(q, kp, vp, bt, ln, st)
        graphs.append((gr, out))
    q.copy_(torch.randn(5, 8, 128, generator=g, device="cuda"))
    ln.copy_(torch.tensor([1500, 803], dtype=torch.int32))
    for gr, out in graphs + graphs:
        with torch.cuda.stream(s):
            gr.replay()
        torch.cuda.current_stream().wait_stream(s)
        check(q, kp, vp, bt, [1500, 803], new, out, None)


def test_cached_tokens_past_32_bit_offsets():
    """A pool of more than 2^32 values: the last pages, read through the table."""
    from fastest_flash_attention_b200 import paged_prefill
    P, page, D = 2 ** 32 // (256 * 128) + 5, 256, 128
    kp, vp = (torch.zeros(P, 1, page, D, device="cuda", dtype=torch.float16) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(0)
    for i in range(P - 3, P):
        for pool in (kp, vp):
            pool[i] = torch.randn(1, page, D, generator=g, device="cuda").half()
    bt = torch.tensor([[P - 1, P - 3, P - 2]], dtype=torch.int32, device="cuda")
    ln = torch.tensor([700], dtype=torch.int32, device="cuda")
    q = torch.randn(10, 4, D, generator=g, device="cuda").half()
    o, lse = paged_prefill(q, kp, vp, bt, ln, starts_of([10]), return_lse=True)
    check(q, kp, vp, bt, [700], [10], o, lse)


def test_nothing_to_do():
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, ln, _ = make([40], 16, 2, 64, torch.float16, 3)
    q = torch.zeros(0, 4, 64, device="cuda", dtype=torch.float16)
    assert paged_prefill(q, kp, vp, bt, ln, starts_of([0])).shape == (0, 4, 64)
    out = torch.full((3, 4, 64), 2.0, device="cuda", dtype=torch.float16)
    assert bool((paged_prefill(out.clone(), kp, vp, bt, ln, starts_of([0]), out=out) == 2).all())
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert bool((paged_prefill(out.clone(), kp, vp, none.view(0, 1), none, starts_of([])[:1], out=out) == 2).all())


@pytest.mark.parametrize("Hq,Hkv,D,softcap,dtype", [
    (28, 4, 128, 30.0, torch.float16),   # seven heads a group: two rows of a tile are nobody's
    (8, 2, 64, None, torch.bfloat16),
    (6, 2, 96, 5.0, torch.bfloat16),
])
def test_a_request_does_not_depend_on_what_shares_its_tile(Hq, Hkv, D, softcap, dtype):
    """The same bits whatever the next request's queries are, and whatever ran before."""
    from fastest_flash_attention_b200 import paged_prefill
    lens, new = [700, 900], [5, 60]
    kp, vp, bt, ln, g = make(lens, 16, Hkv, D, dtype, 31)
    st = starts_of(new)
    q = torch.randn(sum(new), Hq, D, generator=g, device="cuda").to(dtype)
    first = None
    for factor in (1.0, 40.0, 0.0, -300.0, math.nan, 1.0):
        other = q.clone()
        other[new[0]:] *= factor
        o, lse = paged_prefill(other, kp, vp, bt, ln, st, softcap=softcap, return_lse=True)
        if first is None:
            first = o[:new[0]].clone(), lse[:new[0]].clone()
            check(q, kp, vp, bt, lens, new, o, lse, softcap)
        assert torch.equal(o[:new[0]], first[0]) and torch.equal(lse[:new[0]], first[1]), factor
