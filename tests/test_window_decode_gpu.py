"""Paged decode over a sliding window and the first tokens against a plain
64-bit attention over the visible tokens.

Tolerances, derived beforehand.  P is rounded to the data's type (unit roundoff
u: 2^-8 bf16, 2^-11 fp16) and O is rounded to it once; O is a convex combination
of values of magnitude at most V, so |O error| <= 2 u V + fp32 terms.  The fp32
terms: scores up to S in magnitude carry an error of at most (D + 8) 2^-24 S,
which moves O by at most 2 V and the LSE by 1 times as much; 2^x and lg2 are
good to 2^-21.  So |O error| <= V (2 u + 2^-10), |LSE error| <= 2^-10 at the
sizes below (S <= 40, D <= 128)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _make(lens, page, Hkv, D, dtype, window, sinks, seed, freed=True):
    """Pools, a permuted block table whose pages outside window and sinks are -1, lengths."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lens))
    held = [[p for p in range(-(-n // page)) if not freed or p * page < sinks or (p + 1) * page > n - window]
            for n in lens]
    P = max(1, sum(map(len, held)))
    kp, vp = (torch.randn(P, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    ids = torch.randperm(P, generator=g, device="cuda").tolist()
    bt = torch.full((len(lens), width), -1, dtype=torch.int32)
    for r, ps in enumerate(held):
        for p in ps:
            bt[r, p] = ids.pop()
    return kp, vp, bt.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), g


def _check(q, kp, vp, bt, lens, o, lse, window, sinks, softcap=None, scale=None):
    R, Hq, D = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    scale = scale or 1 / math.sqrt(D)
    for r, n in enumerate(lens.tolist()):
        tok = torch.tensor([t for t in range(n) if t >= n - window or t < sinks], device="cuda", dtype=torch.long)
        if n == 0:
            assert bool((o[r] == 0).all()) and bool((lse[r] == -math.inf).all())
            continue
        pg = bt[r, tok // page].long()
        k, v = (x[pg, :, tok % page].double().transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for x in (kp, vp))
        s = (k @ q[r].double()[:, :, None])[..., 0] * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        want = (torch.softmax(s, -1)[:, None] @ v)[:, 0]
        assert float((o[r].double() - want).abs().max()) <= float(v.abs().max()) * (2 * U[q.dtype] + 2.0 ** -10)
        assert float((lse[r].double() - torch.logsumexp(s, -1)).abs().max()) <= 2.0 ** -10


@pytest.mark.parametrize("lens,page,Hq,Hkv,D,window,sinks,softcap,dtype", [
    ([1], 16, 8, 8, 128, 4, 2, None, torch.bfloat16),                       # one token
    ([0, 1, 15, 16, 17, 0, 40], 16, 8, 2, 64, 16, 4, None, torch.float16),  # empty contexts, tile edges
    ([20011], 64, 32, 8, 128, 4096, 4, None, torch.bfloat16),               # a wide cluster
    ([5000, 37, 4096, 4100, 4097], 24, 20, 20, 64, 1000, 1, None, torch.float16),  # pages end inside chunks
    ([300, 999], 5, 7, 1, 96, 250, 13, 30.0, torch.bfloat16),               # tiny pages, head dim 96, softcap
    ([700, 64, 3], 16, 34, 1, 128, 65, 70, None, torch.float16),            # group of 34: three head blocks; sinks > window
    ([130] * 70, 32, 16, 8, 72, 1, 0, None, torch.bfloat16),                # a window of one token, no sinks
    ([513, 2048], 128, 12, 3, 8, 5000, 3, None, torch.float16),             # window past the context, head dim 8
])
def test_window_decode(lens, page, Hq, Hkv, D, window, sinks, softcap, dtype):
    from fastest_flash_attention_b200 import paged_decode
    kp, vp, bt, ln, g = _make(lens, page, Hkv, D, dtype, window, sinks, len(lens) + D)
    q = torch.randn(len(lens), Hq, D, generator=g, device="cuda").to(dtype)
    o, lse = paged_decode(q, kp, vp, bt, ln, sliding_window=window, sink_tokens=sinks, softcap=softcap,
                          return_lse=True)
    _check(q, kp, vp, bt, ln, o, lse, window, sinks, softcap)
    # no LSE, a known longest context (another split), a strided q: the same values to rounding
    wide = torch.zeros(len(lens), Hq, D + 2, device="cuda", dtype=dtype)
    wide[..., 1:D + 1] = q
    o2 = paged_decode(wide[..., 1:D + 1], kp, vp, bt, ln, sliding_window=window, sink_tokens=sinks, softcap=softcap,
                      max_ctx=max(lens))
    _check(q, kp, vp, bt, ln, o2, lse, window, sinks, softcap)


def test_window_decode_is_bit_identical_and_ignores_garbage():
    """Unread rows of the last page and freed pages' entries hold NaN and wild
    ids; two runs give the same bits."""
    from fastest_flash_attention_b200 import paged_decode
    lens, page, window, sinks = [333, 4999, 20], 32, 700, 6
    kp, vp, bt, ln, g = _make(lens, page, 2, 128, torch.bfloat16, window, sinks, 3)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    o, lse = paged_decode(q, kp, vp, bt, ln, sliding_window=window, sink_tokens=sinks, return_lse=True)
    k2, v2, b2 = torch.full_like(kp, math.nan), torch.full_like(vp, math.nan), bt.clone()
    b2[b2 < 0] = 2 ** 30
    for r, n in enumerate(lens):
        tok = torch.tensor([t for t in range(n) if t >= n - window or t < sinks], device="cuda")
        pg = bt[r, tok // page].long()
        k2[pg, :, tok % page], v2[pg, :, tok % page] = kp[pg, :, tok % page], vp[pg, :, tok % page]
    o2, lse2 = paged_decode(q, k2, v2, b2, ln, sliding_window=window, sink_tokens=sinks, return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_window_decode_with_all_visible_matches_the_plain_decode():
    from fastest_flash_attention_b200 import paged_decode
    kp, vp, bt, ln, g = _make([700, 64, 1], 16, 2, 128, torch.float16, 700, 0, 5)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(torch.float16)
    o, lse = paged_decode(q, kp, vp, bt, ln, sliding_window=700, return_lse=True)
    o2, lse2 = paged_decode(q, kp, vp, bt, ln, return_lse=True, sink_tokens=3)  # no window: every token
    V = float(vp.abs().max())
    assert float((o.double() - o2.double()).abs().max()) <= 2 * V * (2 * U[torch.float16] + 2.0 ** -10)
    assert float((lse - lse2).abs().max()) <= 2 * 2.0 ** -10


def test_window_decode_refusals():
    from fastest_flash_attention_b200 import paged_decode
    kp, vp, bt, ln, g = _make([40], 16, 2, 64, torch.float16, 40, 0, 1)
    q = torch.randn(1, 4, 64, device="cuda", dtype=torch.float16)
    for kw in (dict(sliding_window=-1), dict(sliding_window=4, sink_tokens=-1), dict(sink_tokens=-2)):
        with pytest.raises(ValueError):
            paged_decode(q, kp, vp, bt, ln, **kw)
    for bad in ((q.float(), kp, vp, bt, ln), (q[:, :3], kp, vp, bt, ln), (q[..., :8], kp, vp, bt, ln),
                (q, kp, vp[:, :1], bt, ln), (q, kp.transpose(2, 3), vp.transpose(2, 3), bt, ln), (q, kp, vp, bt[0], ln),
                (q, kp, vp, bt, ln[:0]), (q[0], kp, vp, bt, ln)):
        with pytest.raises(ValueError):
            paged_decode(*bad, sliding_window=16)
    wide = torch.zeros(2, 2, 16, 136, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        paged_decode(torch.zeros(1, 4, 136, device="cuda", dtype=torch.float16), wide, wide, bt, ln, sliding_window=16)
    for lens, table, word in ((torch.full_like(ln, 49), bt, "context length"), (ln, bt * 0 + 99, "block-table entry")):
        with pytest.raises(RuntimeError, match=word):
            paged_decode(q, kp, vp, table, lens, sliding_window=16)


def test_cache_decode_after_trim_fork_and_compact():
    """The windowed decode of a cache is the same before and after its pages
    outside the window are freed, in a fork, and after compaction."""
    from fastest_flash_attention_b200 import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(2)
    c = PagedKVCache(max_pages=300, page_size=16, num_heads=2, head_dim=128, dtype=torch.bfloat16, device="cuda")
    for s, n in enumerate((900, 77, 1500)):
        k, v = (torch.randn(2, n, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        c.append_tokens(s, k, v)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    kw = dict(sliding_window=256, sink_tokens=4)
    want = c.decode(q, [0, 1, 2], **kw)
    for s in (0, 2):
        assert c.trim_sequence(s, 256, 4) > 0
    assert torch.equal(c.decode(q, [0, 1, 2], **kw), want)
    c.fork_sequence(2, 9)
    assert torch.equal(c.decode(q, [0, 1, 9], **kw), want)
    assert c.compact_sequences([0, 1, 9], 256, 4) == 900 - 260 + 1500 - 260
    assert torch.equal(c.decode(q, [0, 1, 9], **kw), want) and torch.equal(c.decode(q, [0, 1, 2], **kw), want)
