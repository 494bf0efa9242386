"""Decoding behind shared prefixes against a plain 64-bit attention of each
request.

Tolerances, derived beforehand, as test_paged_prefill_gpu.py's: P rounded to the
data's type (unit roundoff u) and O rounded once more, 2 u V for values up to V;
the fp32 terms (scores, 2^x, the join of partial results, whose weights sum to 1)
within 2^-10 V.  LSE 2^-10."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(groups, alone, page, Hkv, D, dtype, seed):
    """groups: [(prefix tokens, [tokens behind it of each member])], alone: lengths.  Full pages of a prefix are
    shared, the page that it ends in is each member's own copy; the first member lends its row.  What no request
    reads is NaN (pools) or -1 (table)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, starts, prefixes, rows = [], [0], [], []
    pages = 0
    for n, own in groups:
        first = None
        for x in own:
            full = n // page if first is not None else 0
            count = max(-(-(n + x) // page), 0) - full
            rows.append((first[:full] if first is not None else []) + list(range(pages, pages + count)))
            pages += count
            first = first if first is not None else rows[-1]
            lens.append(n + x)
        starts.append(len(lens))
        prefixes.append(n)
    for x in alone:
        rows.append(list(range(pages, pages + -(-x // page))))
        pages += -(-x // page)
        lens.append(x)
    P = pages + 2
    perm = torch.randperm(P, generator=g, device="cuda").tolist()
    bt = torch.full((len(lens), max(1, max(map(len, rows)))), -1, dtype=torch.int32)
    for r, ids in enumerate(rows):
        bt[r, :len(ids)] = torch.tensor([perm[i] for i in ids], dtype=torch.int32)
    bt = bt.cuda()
    kp, vp = (torch.full((P, Hkv, page, D), math.nan, device="cuda", dtype=dtype) for _ in range(2))

    def write(r, a, b, like=None):
        tok = torch.arange(a, b, device="cuda")
        for pool in (kp, vp):
            x = torch.randn(b - a, Hkv, D, generator=g, device="cuda").to(dtype) if like is None \
                else pool[bt[like, tok // page].long(), :, tok % page]
            pool[bt[r, tok // page].long(), :, tok % page] = x
    for i, (n, own) in enumerate(groups):
        for r in range(starts[i], starts[i + 1]):
            if r == starts[i]:
                write(r, 0, n)
            else:
                write(r, n // page * page, n, like=starts[i])
            write(r, n, lens[r])
    for r in range(starts[-1], len(lens)):
        write(r, 0, lens[r])

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    return kp, vp, bt, ints(lens), ints(starts), ints(prefixes), g


def check(q, kp, vp, bt, lens, o, lse, softcap=None, scale=None, rows=None):
    R, Hq, D = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    for r, n in enumerate(lens.tolist()):
        if rows is not None and r not in rows:
            continue
        if n == 0:
            assert bool((o[r] == 0).all()) and (lse is None or bool((lse[r] == -math.inf).all()))
            continue
        tok = torch.arange(n, device="cuda")
        pg = bt[r, tok // page].long()
        k, v = (x[pg, :, tok % page].double().transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for x in (kp, vp))
        s = (k @ q[r].double()[:, :, None])[..., 0] * (scale or 1 / math.sqrt(D))
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        want = (torch.softmax(s, -1)[:, None] @ v)[:, 0]
        assert float((o[r].double() - want).abs().max()) <= float(v.abs().max()) * (2 * U[q.dtype] + 2.0 ** -10), r
        if lse is not None:
            assert float((lse[r].double() - torch.logsumexp(s, -1)).abs().max()) <= 2.0 ** -10, r


CASES = [
    # groups, alone, page, Hq, Hkv, D, softcap, dtype
    ([(1, [0])], [], 16, 1, 1, 64, None, torch.bfloat16),                                # one token, one request
    ([(200, [1, 40, 7, 0])], [], 16, 8, 2, 64, None, torch.float16),
    ([(16, [1, 2]), (128, [1] * 5), (129, [0, 3])], [0, 5, 200], 16, 4, 4, 128, None, torch.bfloat16),  # tile edges
    ([(77, [3] * 20), (4099, [0, 333] * 4), (1000, [5])], [0, 17], 24, 21, 3, 96, 30.0, torch.float16),
    ([(5000, list(range(1, 65)))], [], 64, 32, 8, 128, None, torch.bfloat16),            # two tiles a kv head, split
    ([(3001, [900, 1, 0])], [], 128, 8, 1, 128, None, torch.float16),                    # one kv head, a wide split
    ([(500, [2] * 130)], [], 8, 3, 3, 72, 2.0, torch.bfloat16),                          # no grouping, a tight cap
    ([(300, [1, 2])], [40], 40, 128, 1, 8, None, torch.float16),                         # group of 128, head dim 8
    ([(8 * (i + 1), [i % 3, 1]) for i in range(40)], [9], 8, 4, 2, 64, None, torch.float16),  # more groups than lanes
    ([(0, [5, 6]), (64, [])], [3], 16, 4, 2, 64, None, torch.bfloat16),                  # nothing shared; no members
]


@pytest.mark.parametrize("groups,alone,page,Hq,Hkv,D,softcap,dtype", CASES)
def test_prefix_decode(groups, alone, page, Hq, Hkv, D, softcap, dtype):
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make(groups, alone, page, Hkv, D, dtype, len(groups) + D)
    R = ln.shape[0]
    q = torch.randn(R, Hq, D, generator=g, device="cuda").to(dtype)
    o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, softcap=softcap, return_lse=True)
    check(q, kp, vp, bt, ln, o, lse, softcap)
    wide = torch.full((R, Hq, D + 8), math.nan, device="cuda", dtype=dtype)
    wide[..., :D] = q
    top = int(pf.max())
    for hints in (dict(max_prefix=1, max_own=1), dict(max_prefix=top, max_own=max(1, int(ln.max()))),
                  dict(max_prefix=50 * top)):
        o2 = prefix_decode(wide[..., :D], kp, vp, bt.long(), ln.long(), st.long(), pf.long(), softcap=softcap,
                           scale=0.3, **hints)
        check(q, kp, vp, bt, ln, o2, None, softcap, 0.3)


def test_without_groups():
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([], [0, 100, 33], 16, 2, 64, torch.float16, 1)
    q = torch.randn(3, 8, 64, generator=g, device="cuda").half()
    o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, return_lse=True)
    check(q, kp, vp, bt, ln, o, lse)
    none = q[:0]
    assert prefix_decode(none, kp, vp, bt[:0], ln[:0], st, pf).shape == (0, 8, 64)


def test_members_shorter_than_the_prefix():
    """They share nothing, and lend nothing: their rows hold other pages, or none."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([], [10, 0, 150, 150, 63], 16, 2, 128, torch.bfloat16, 2)
    bt[3, :4] = bt[2, :4]  # requests 2 and 3 share 64 tokens; 0, 1 and 4 lie in their group
    for start, end in ((0, 5), (1, 4), (2, 4)):
        st = torch.tensor([start, end], dtype=torch.int32, device="cuda")
        pf = torch.tensor([64], dtype=torch.int32, device="cuda")
        q = torch.randn(5, 8, 128, generator=g, device="cuda").bfloat16()
        o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, return_lse=True)
        check(q, kp, vp, bt, ln, o, lse)


def test_same_bits_and_same_as_the_plain_decode():
    from fastest_flash_attention_b200 import paged_decode, prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(1000, [5, 300, 1, 64])], [], 16, 2, 128, torch.bfloat16, 3)
    q = torch.randn(4, 8, 128, generator=g, device="cuda").bfloat16()
    a, b = (prefix_decode(q, kp, vp, bt, ln, st, pf, return_lse=True) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    kp.nan_to_num_(0.0)
    vp.nan_to_num_(0.0)
    bt.clamp_(min=0)
    o, lse = paged_decode(q, kp, vp, bt, ln, return_lse=True)
    V = float(vp.abs().max())
    assert float((a[0].double() - o.double()).abs().max()) <= 2 * V * (2 * U[torch.bfloat16] + 2.0 ** -10)
    assert float((a[1] - lse).abs().max()) <= 2 * 2.0 ** -10


def test_data_that_means_nothing_is_reported():
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(64, [3, 5])], [7], 16, 2, 64, torch.float16, 4)
    q = torch.randn(3, 8, 64, generator=g, device="cuda").half()

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    for kw, word in ((dict(st=ints(0, 4)), "boundaries"), (dict(st=ints(2, 1)), "boundaries"),
                     (dict(st=ints(-1, 2)), "boundaries"), (dict(pf=ints(-1)), "prefix"),
                     (dict(pf=ints(1000)), "prefix"), (dict(ln=ints(67, -2, 7)), "context length"),
                     (dict(ln=ints(67, 900, 7)), "context length"), (dict(bt=bt * 0 + 99), "block-table entry"),
                     (dict(bt=bt * 0 - 1), "block-table entry"), (dict(pf=pf.long() + 2 ** 32), "prefix"),
                     (dict(st=st.long() + 2 ** 32), "boundaries")):
        a = dict(dict(bt=bt, ln=ln, st=st, pf=pf), **kw)
        with pytest.raises(RuntimeError, match=word):
            prefix_decode(q, kp, vp, a["bt"], a["ln"], a["st"], a["pf"])
    o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, return_lse=True)
    check(q, kp, vp, bt, ln, o, lse)


def test_captured_and_replayed_on_a_side_stream():
    """Two graphs of one call, replayed with other contents (another grouping among them), on a stream of their own."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(2000, [5, 300, 1, 64])], [70], 16, 2, 128, torch.bfloat16, 3)
    q = torch.randn(5, 8, 128, generator=g, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        prefix_decode(q, kp, vp, bt, ln, st, pf, max_prefix=2000, max_own=300)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = prefix_decode(q, kp, vp, bt, ln, st, pf, max_prefix=2000, max_own=300)
        graphs.append((gr, out))
    for starts, prefix in (([0, 4], 2000), ([1, 3], 1600), ([0, 5], 1999), ([5, 5], 2000)):
        st.copy_(torch.tensor(starts))
        pf.fill_(prefix)
        q.copy_(torch.randn(5, 8, 128, generator=g, device="cuda"))
        for gr, out in graphs:
            with torch.cuda.stream(s):
                s.wait_stream(torch.cuda.default_stream())
                gr.replay()
            torch.cuda.current_stream().wait_stream(s)
            check(q, kp, vp, bt, ln, out, None)


def test_calls_in_a_row_wait_for_each_other(monkeypatch):
    """Launches that overlap: many calls behind one another, each reading what the call before wrote."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(900, [5, 30, 1, 64])], [], 16, 8, 128, torch.bfloat16, 6)
    q = torch.randn(4, 8, 128, generator=g, device="cuda").bfloat16()
    monkeypatch.setenv("FFA_SYNC_CHECK", "0")
    chain = [q]
    for _ in range(30):
        chain.append(prefix_decode(chain[-1], kp, vp, bt, ln, st, pf))
    for a, b in zip(chain[::7], chain[1::7]):
        check(a, kp, vp, bt, ln, b, None)


@pytest.mark.parametrize("groups,alone,page,Hq,Hkv,D,softcap,dtype", [
    ([(20000, [3, 0, 40] * 13)], [0, 30], 16, 8, 4, 64, None, torch.float16),
    ([(12000, [1, 17] * 80)], [5] * 9, 40, 2, 1, 96, 20.0, torch.bfloat16),
    ([(9000, [i % 50 for i in range(150)]), (0, [4, 4]), (4001, [0])], [], 64, 8, 2, 128, None, torch.bfloat16),
])
def test_own_tokens_beside_a_long_prefix(groups, alone, page, Hq, Hkv, D, softcap, dtype):
    """Shapes whose own tokens are partial results too, joined by a third launch; eager, captured, on unshared rows."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make(groups, alone, page, Hkv, D, dtype, 11)
    R = ln.shape[0]
    q = torch.randn(R, Hq, D, generator=g, device="cuda").to(dtype)
    top = int(pf.max())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = prefix_decode(q, kp, vp, bt, ln, st, pf, softcap=softcap, return_lse=True, max_prefix=top, max_own=50)
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        b = prefix_decode(q, kp, vp, bt, ln, st, pf, softcap=softcap, return_lse=True, max_prefix=top, max_own=50)
        c = b[0] + 0  # what follows the call in a graph sees all of it
    for t in b:
        t.fill_(math.nan)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[0], c)
    check(q, kp, vp, bt, ln, a[0], a[1], softcap)
    top = bt.shape[1] * page  # nobody is as long: each request by itself
    assert top > int(ln.max())
    o = prefix_decode(q, kp, vp, bt, ln, st, pf * 0 + top, softcap=softcap, max_prefix=top, max_own=top)
    check(q, kp, vp, bt, ln, o, None, softcap, rows=range(0, R, 7))


def padded(bt, tokens, page):
    """bt with columns for `tokens` tokens, which lets max_prefix say anything."""
    wide = torch.full((bt.shape[0], tokens // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :bt.shape[1]] = bt
    return wide


@pytest.mark.parametrize("groups,alone,page,Hq,Hkv,D,softcap,dtype", CASES + [
    ([(128, [1, 0] * 50), (129, [3] * 60), (40, [2] * 40)], [5], 16, 32, 8, 128, None, torch.bfloat16),
    ([(77, [i % 9 for i in range(90)]), (256, [0] * 70)], [1, 0], 8, 40, 8, 96, 5.0, torch.float16),
])
def test_prefix_for_the_group_or_for_each_request(groups, alone, page, Hq, Hkv, D, softcap, dtype):
    """Either way that the sizes may choose, eager and in a graph; the prefix is read through the group's first row."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make(groups, alone, page, Hkv, D, dtype, 5)
    q = torch.randn(ln.shape[0], Hq, D, generator=g, device="cuda").to(dtype)
    lent = padded(bt, 65536, page)
    for i, (n, own) in enumerate(groups):
        lent[sum(len(x) for _, x in groups[:i]) + 1:sum(len(x) for _, x in groups[:i + 1]), :n // page] = -1
    for hint in (1, 65536):
        args = (q, kp, vp, lent, ln, st, pf)
        kw = dict(softcap=softcap, return_lse=True, max_prefix=hint, max_own=50)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            a = prefix_decode(*args, **kw)
        torch.cuda.current_stream().wait_stream(s)
        check(q, kp, vp, bt, ln, a[0], a[1], softcap)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            b = prefix_decode(*args, **kw)
        for _ in range(2):
            for t in b:
                t.fill_(math.nan)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("hint", [1, 65536])
def test_data_that_means_nothing_is_reported_either_way(hint):
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(64, [3, 5]), (32, [1])], [7], 16, 2, 64, torch.float16, 4)
    q = torch.randn(4, 8, 64, generator=g, device="cuda").half()
    bt = padded(bt, 65536, 16)

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    for kw, word in ((dict(st=ints(0, 2, 5)), "boundaries"), (dict(st=ints(0, 3, 1)), "boundaries"),
                     (dict(st=ints(-2 ** 31, 2, 3)), "boundaries"), (dict(pf=ints(64, -1)), "prefix"),
                     (dict(pf=ints(2 ** 31 - 1, 32)), "prefix"), (dict(ln=ints(67, 65537, 33, 7)), "context length"),
                     (dict(ln=ints(67, 69, -1, 7)), "context length"), (dict(bt=bt * 0 + 99), "block-table entry")):
        a = dict(dict(bt=bt, ln=ln, st=st, pf=pf), **kw)
        with pytest.raises(RuntimeError, match=word):
            prefix_decode(q, kp, vp, a["bt"], a["ln"], a["st"], a["pf"], max_prefix=hint)
    o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, return_lse=True, max_prefix=hint)
    check(q, kp, vp, bt, ln, o, lse)


@pytest.mark.parametrize("own", [0, 1])
def test_softcap_of_few_small_scores(own):
    """LSEs of one and two tokens to 16 fp32 roundings of the larger of 1 and the score (the product, the scale, the
    cap, the logarithm's parts), and not to an absolute error that grows with the cap."""
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make([(1, [own] * 9)], [], 16, 1, 64, torch.float16, 8)
    q = (torch.randn(9, 4, 64, generator=g, device="cuda") / 4).half()
    for cap in (30.0, 300.0):
        _, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, softcap=cap, return_lse=True)
        tok = torch.arange(1 + own, device="cuda")
        k = kp[bt[:, tok // 16].long(), 0, tok % 16].double()
        s = cap * torch.tanh((q.double() @ k.transpose(1, 2)) / 8 / cap)
        bound = 16 * 2.0 ** -24 * s.abs().amax(-1).clamp(min=1.0)
        assert bool(((lse.double() - torch.logsumexp(s, -1)).abs() <= bound).all())
