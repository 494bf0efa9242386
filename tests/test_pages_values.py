"""Values of attention over pages, closely enough that a wrong page of V shows in the
longest contexts.  O of n random keys shrinks as 1 / sqrt(n), so an absolute bound, or
one by the largest value, lets a page pass there (and the LSE knows nothing of V).  Here
the error's norm over a row's D columns is held against what rounding can make of it.

Derived beforehand.  u: half a step of the data's type (2^-8 bf16, 2^-11 fp16), p_j the
row's weights, v_j its values, W = sqrt(sum p_j^2 |v_j|^2), R the largest norm of the
sum of p_j v_j over any first tokens.
  - O is rounded once: u |o|.
  - each p_j is rounded once, by errors of at most u p_j and of either sign: their
    sum's norm has a mean square of at most u^2 W^2 / 3; 2 u W is 3.4 times its root,
    and more than any error of up to four keys.
  - scores carry (D + 8) 2^-24 S at most, S the largest scale * sum |q_d k_d| (with a
    cap, which only shrinks them, its own 2^-21 cap more), and 2^x 2^-18: relative
    errors of p of either sign again, within 8 W of their sum, and of the row's sum,
    which divides all alike: 2 |o| of it, with the fp32 sum's own n 2^-26.
  - the tensor core cuts a product off some 25 bits below the sum that it joins: n
    products, 2^-24 of at most 2 R.
  - fp16 P below 2^-14 of its largest is off by 2^-25 of that: 2^-25 sum |v_j| / l, l
    the sum of e^(s_j - max).
The LSE: the scores' error, 2^-17, n 2^-26, and its fp32 rounding."""
import math

import pytest
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def attend(q, k, v, limits, scale, softcap=None):
    """64-bit (o, lse, o's tolerance, lse's) of rows q [m, D] over the first limits[i] >= 1 of k, v [n, D]; q, k, v in
    their 16-bit type."""
    dtype, D, n = q.dtype, q.shape[1], k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    s = q @ k.T * scale
    ds = (D + 8) * 2.0 ** -24 * (q.abs() @ k.abs().T * scale)
    if softcap:
        s, ds = softcap * torch.tanh(s / softcap), ds + 2.0 ** -21 * softcap
    hide = torch.arange(n, device=q.device)[None, :] >= limits[:, None]
    s, ds = s.masked_fill(hide, -math.inf), ds.masked_fill(hide, 0).amax(1)
    p, lse = torch.softmax(s, 1), torch.logsumexp(s, 1)
    o = p @ v
    v2 = (v * v).sum(1)
    W = (p * p @ v2).sqrt()
    tiles = -(-n // 64)
    pt = torch.nn.functional.pad(p, (0, tiles * 64 - n)).view(-1, tiles, 64)
    vt = torch.nn.functional.pad(v, (0, 0, 0, tiles * 64 - n)).view(tiles, 64, D)
    R = torch.einsum("mtj,tjd->mtd", pt, vt).cumsum(1).norm(dim=2).amax(1) + W
    rel = ds + 2.0 ** -18
    norm = o.norm(dim=1)
    tol = U[dtype] * norm + (2 * U[dtype] + 8 * rel) * W + (2 * rel + n * 2.0 ** -26) * norm + n * 2.0 ** -23 * R
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25 * v2.sqrt().sum() / torch.exp(s - s.amax(1, keepdim=True)).sum(1)
    return o, lse, tol, rel + 2.0 ** -17 + n * 2.0 ** -26 + 2.0 ** -22 * lse.abs(), p


def worst(o, q, k, v, limits, scale, softcap=None, lse=None):
    """The largest error of a row's O (and LSE) in units of its tolerance."""
    want, wl, tol, tl, _ = attend(q, k, v, limits, scale, softcap)
    far = float(((o.double() - want).norm(dim=1) / tol).max())
    return far if lse is None else max(far, float(((lse.double() - wl).abs() / tl).max()))


# ------------------------------------------------------------------- the bound itself, on the CPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3, 40, 300, 2500, 5000, 9000, 12000, 20000])
def test_the_bound_passes_rounding_and_no_wrong_page(n, dtype):
    """O from weights and values rounded as a kernel rounds them lies within it; O with a page of 16 tokens whose
    values are another page's, or are left out, lies outside, wherever the page is."""
    g = torch.Generator().manual_seed(n)
    D, m = 64, 4
    q, k, v = (torch.randn(r, D, generator=g).to(dtype) for r in (m, n, n))
    limits = torch.full((m,), n)
    _, lse, _, _, p = attend(q, k, v, limits, 1 / math.sqrt(D))
    top = p.amax(1, keepdim=True)
    rounded = (p / top).to(dtype).double() * top
    assert worst((rounded @ v.double()).to(dtype), q, k, v, limits, 1 / math.sqrt(D), lse=lse.float()) <= 1
    if n < 40:
        return
    for at in sorted({0, 16, n // 2 // 16 * 16, (n - 16) // 16 * 16}):
        other = (at + 16 + n // 3 // 16 * 16) % (n // 16 * 16)
        assert other != at
        for page in (v[other:other + 16], torch.zeros(16, D, dtype=dtype)):
            wrong = v.clone()
            wrong[at:at + 16] = page
            o = (rounded @ wrong.double()).to(dtype)
            far = (o.double() - p @ v.double()).norm(dim=1) / attend(q, k, v, limits, 1 / math.sqrt(D))[2]
            assert float(far.max()) > 1, (at, far)  # (the largest row is what a test asserts)


# ------------------------------------------------------------------------------------- the kernels
def check(q, kp, vp, bt, r, n, past, o, lse, softcap, scale=None):
    """q [m, Hq, D] of request r over its n tokens, query i over the first past + i + 1."""
    m, Hq, D = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    tok = torch.arange(n, device="cuda")
    pg = bt[r].long()[tok // page]
    limits = past + torch.arange(m, device="cuda") + 1
    group, step = Hq // Hkv, max(1, (1 << 24) // n)
    for h in range(Hkv):
        k, v = (x[pg, h, tok % page] for x in (kp, vp))
        heads = slice(h * group, (h + 1) * group)
        rows = [x[:, heads].reshape(m * group, *x.shape[2:]) for x in (q, o)]
        lim, ls = limits.repeat_interleave(group), lse[:, heads].reshape(-1)
        for a in range(0, m * group, step):
            b = slice(a, a + step)
            far = worst(rows[1][b], rows[0][b], k, v, lim[b], scale or 1 / math.sqrt(D), softcap, ls[b])
            assert far <= 1, (r, h, a, far)


PREFILL = [
    # lens, new, page, Hq, Hkv, D, softcap, dtype
    ([2500], [3], 64, 32, 8, 128, None, torch.bfloat16),
    ([5000, 3, 4000], [1, 2, 300], 128, 8, 1, 128, None, torch.float16),
    ([6000], [1500], 16, 4, 1, 64, None, torch.bfloat16),
    ([12000, 9000], [4, 2], 16, 8, 2, 128, None, torch.bfloat16),
    ([20000, 700], [2, 700], 24, 6, 2, 64, 30.0, torch.float16),
    ([9000], [300], 40, 7, 1, 96, 20.0, torch.bfloat16),
    ([900 + i for i in range(40)], [(i * 29) % 90 for i in range(40)], 64, 8, 2, 128, None, torch.bfloat16),
    ([127, 1, 0, 333], [127, 1, 0, 64], 8, 4, 4, 72, None, torch.float16),
    ([400, 20], [9, 20], 40, 128, 1, 8, None, torch.float16),
    # lopsided: one long context among short ones, a chunk beside single tokens
    ([40000] + [900] * 70, [4] * 71, 64, 8, 2, 128, None, torch.bfloat16),
    ([1] * 40 + [8512] + [1000] * 30, [1] * 40 + [512] + [1] * 30, 16, 4, 1, 128, None, torch.float16),
    ([20, 30000, 17], [20, 1, 3], 24, 5, 5, 64, None, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hint", ["none", "short", "exact", "long"])
@pytest.mark.parametrize("lens,new,page,Hq,Hkv,D,softcap,dtype", PREFILL)
def test_prefill(lens, new, page, Hq, Hkv, D, softcap, dtype, hint):
    from test_paged_prefill_gpu import make, starts_of
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, ln, g = make(lens, page, Hkv, D, dtype, 50 + len(lens) + D)
    q = torch.randn(sum(new), Hq, D, generator=g, device="cuda").to(dtype)
    o, lse = paged_prefill(q, kp, vp, bt, ln, starts_of(new), softcap=softcap, return_lse=True,
                           max_ctx={"none": None, "short": 1, "exact": max(lens), "long": 40 * max(lens)}[hint])
    at = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        if m:
            check(q[at:at + m], kp, vp, bt, r, n, n - m, o[at:at + m], lse[at:at + m], softcap)
        at += m


PREFIX = [
    # groups, alone, page, Hq, Hkv, D, softcap, dtype
    ([(200, [1, 40, 7, 0])], [], 16, 8, 2, 64, None, torch.float16),
    ([(16, [1, 2]), (128, [1] * 5), (129, [0, 3])], [5, 200], 16, 4, 4, 128, None, torch.bfloat16),
    ([(77, [3] * 20), (4099, [0, 333] * 4), (1000, [5])], [17], 24, 21, 3, 96, 30.0, torch.float16),
    ([(5000, list(range(1, 65)))], [], 64, 32, 8, 128, None, torch.bfloat16),
    ([(3001, [900, 1, 0])], [9000], 128, 8, 1, 128, None, torch.float16),
    ([(20000, [3, 0, 40] * 13)], [30], 16, 8, 4, 64, None, torch.float16),
    ([(12000, [1, 17] * 80)], [5] * 9, 40, 2, 1, 96, 20.0, torch.bfloat16),
    ([(9000, [i % 50 for i in range(150)]), (4001, [0])], [], 64, 8, 2, 128, None, torch.bfloat16),
    ([(8192, [1 + 97 * i % 1024 for i in range(24)])], [], 16, 8, 2, 128, None, torch.bfloat16),
    # lopsided: a long request that shares nothing, one long among a group's own tokens, groups of 1 and 60
    ([(960, [40] * 40)], [30000], 64, 8, 2, 128, None, torch.bfloat16),
    ([(128, [3] * 9 + [20000] + [0] * 20)], [], 16, 4, 4, 64, None, torch.float16),
    ([(9000, [5]), (40, [i % 7 for i in range(60)])], [1], 8, 16, 2, 96, None, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hint", ["none", "short", "exact"])
@pytest.mark.parametrize("groups,alone,page,Hq,Hkv,D,softcap,dtype", PREFIX)
def test_prefix_decode(groups, alone, page, Hq, Hkv, D, softcap, dtype, hint):
    from test_prefix_decode_gpu import make
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, ln, st, pf, g = make(groups, alone, page, Hkv, D, dtype, 60 + len(groups) + D)
    R = ln.shape[0]
    q = torch.randn(R, Hq, D, generator=g, device="cuda").to(dtype)
    own = max([x for _, mine in groups for x in mine] + alone)
    hints = {"none": {}, "short": dict(max_prefix=1, max_own=1), "exact": dict(max_prefix=int(pf.max()), max_own=own)}
    o, lse = prefix_decode(q, kp, vp, bt, ln, st, pf, softcap=softcap, return_lse=True, **hints[hint])
    for r in sorted({*range(min(R, 12)), *range(12, R, 11), R - 1}):
        check(q[r:r + 1], kp, vp, bt, r, int(ln[r]), int(ln[r]) - 1, o[r:r + 1], lse[r:r + 1], softcap)
