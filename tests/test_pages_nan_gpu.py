"""Query rows over pages where a visible key is NaN, or its score +inf: the row's
softmax is NaN, whichever column of a key tile the key lies in, and the LSE says
so too (NaN; +inf where an infinite score is all that is wrong), so that no later
join by LSE takes the row for an ordinary one.  Rows that do not see the key stay
as they are: within twice the tolerance of test_paged_prefill_gpu.py of a clean
run, each run being within one of the exact values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pools(R, n, page, Hkv, D, dtype, seed):
    """R rows of n tokens in pages of their own, in random order; the rows' pages [R, ceil(n / page)]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-n // page)
    bt = torch.randperm(R * per, generator=g, device="cuda").view(R, per).int()
    kp, vp = (torch.randn(R * per, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    return kp, vp, bt, g


def plant(kp, bt, rows, toks, page, what):
    """Token toks[i] of row rows[i] becomes NaN, or infinite in its first column (queries are positive there)."""
    kp = kp.clone()
    pg, off = bt[rows, toks // page].long(), toks % page
    if what == "nan":
        kp[pg, :, off] = math.nan
    else:
        kp[pg, :, off, 0] = math.inf
    return kp


def query(T, Hq, D, g, dtype):
    q = torch.randn(T, Hq, D, generator=g, device="cuda")
    q[..., 0] = q[..., 0].abs() + 1
    return q.to(dtype)


def poisoned(o, lse):
    return o.isnan().all(-1) & (lse.isnan() | (lse == math.inf))


# R, tokens, new, page, Hq, Hkv, D, dtype: one tile at D 64; 32 rows; one tile of 128 rows; two of them
FORMS = [(192, 192, 1, 16, 4, 2, 64, torch.bfloat16), (256, 256, 2, 24, 8, 2, 128, torch.float16),
         (256, 256, 40, 64, 2, 2, 96, torch.bfloat16), (256, 256, 150, 16, 1, 1, 128, torch.bfloat16),
         (192, 192, 100, 8, 3, 1, 64, torch.float16)]


@pytest.mark.parametrize("softcap", [None, 20.0])
@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("R,n,new,page,Hq,Hkv,D,dtype", FORMS)
def test_every_column_of_a_tile(R, n, new, page, Hq, Hkv, D, dtype, what, softcap):
    """Request r's token r is the one: every column of the first tiles."""
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, g = pools(R, n, page, Hkv, D, dtype, D + new)
    q = query(R * new, Hq, D, g, dtype)
    args = (bt, ints([n] * R), ints([new * r for r in range(R + 1)]))
    rows = torch.arange(R, device="cuda")
    clean, clean_lse = paged_prefill(q, kp, vp, *args, return_lse=True, softcap=softcap)
    o, lse = paged_prefill(q, plant(kp, bt, rows, rows, page, what), vp, *args, return_lse=True, softcap=softcap)
    sees = (n - new + torch.arange(new, device="cuda")[None, :] >= rows[:, None]).reshape(-1)
    if what == "nan" or not softcap:
        assert bool(poisoned(o, lse)[sees].all())
    else:  # a cap makes an infinite score a large one
        assert bool(o.isfinite().all() and lse.isfinite().all())
    other = ~sees
    assert bool(other.any()) == (new > 1)
    bound = 2 * float(vp.abs().max()) * (2 * U[dtype] + 2.0 ** -10)
    assert bool(((o - clean).double().abs() <= bound)[other].all())
    assert bool(((lse - clean_lse).abs() <= 2 * 2.0 ** -10)[other].all())


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("page,Hq,Hkv,D,dtype", [(64, 32, 8, 128, torch.bfloat16), (16, 8, 1, 64, torch.float16)])
def test_shares_of_a_long_context(page, Hq, Hkv, D, dtype, what):
    """A context that is cut: the partial results' join keeps it."""
    from fastest_flash_attention_b200 import paged_prefill
    n, new = 6000, 3
    kp, vp, bt, g = pools(1, n, page, Hkv, D, dtype, 2)
    q = query(new, Hq, D, g, dtype)
    row = torch.zeros(1, dtype=torch.int64, device="cuda")
    for tok in list(range(0, 64)) + [127, 128, 1000, 2506, 5990, 5997]:
        bad = plant(kp, bt, row, row + tok, page, what)
        o, lse = paged_prefill(q, bad, vp, bt, ints([n]), ints([0, new]), return_lse=True)
        assert bool(poisoned(o, lse).all()), tok


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("hint", [1, 65536])
@pytest.mark.parametrize("page,Hq,Hkv,D,dtype", [(16, 8, 2, 128, torch.bfloat16), (8, 4, 4, 64, torch.float16)])
def test_every_column_of_a_shared_prefix(page, Hq, Hkv, D, dtype, hint, what):
    """Groups of two behind prefixes of 128 tokens, token i of group i's the one; by either way of reading it."""
    from fastest_flash_attention_b200 import prefix_decode
    G, n = 128, 128
    kp, vp, own, g = pools(2 * G, n + page, page, Hkv, D, dtype, 7)
    own[1::2, :n // page] = own[::2, :n // page]
    bt = torch.full((2 * G, 65536 // page), -1, dtype=torch.int32, device="cuda")
    bt[:, :own.shape[1]] = own
    q = query(2 * G, Hq, D, g, dtype)
    rows = torch.arange(G, device="cuda")
    for keep in (False, True):  # and a second time where only every other group has one
        some = rows[1::2] if keep else rows
        bad = plant(kp, bt, 2 * some, some, page, what)
        o, lse = prefix_decode(q, bad, vp, bt, ints([n + 3] * (2 * G)), ints(list(range(0, 2 * G + 1, 2))),
                               ints([n] * G), return_lse=True, max_prefix=hint, max_own=page)
        hit = torch.zeros(G, dtype=torch.bool, device="cuda")
        hit[some] = True
        hit = hit.repeat_interleave(2)
        assert bool(poisoned(o, lse)[hit].all())
        assert bool(o[~hit].isfinite().all() and lse[~hit].isfinite().all())


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_joins_of_a_long_prefix(where, what):
    """Shares of the prefix, and own tokens that are a partial result themselves (a third launch)."""
    from fastest_flash_attention_b200 import prefix_decode
    n, R, page, own = 20000, 40, 16, 64
    kp, vp, bt, g = pools(R, n // R + own, page, 4, 64, torch.float16, 3)  # (as many pages as are needed)
    ids = bt.reshape(-1)
    bt = torch.empty(R, (n + own) // page, dtype=torch.int32, device="cuda")
    bt[:, :n // page] = ids[:n // page]
    bt[:, n // page:] = ids[n // page:n // page + R * (own // page)].view(R, -1)
    q = query(R, 8, 64, g, torch.float16)
    lens = ints([n + 1 + i for i in range(R)])
    clean = prefix_decode(q, kp, vp, bt, lens, ints([0, R]), ints([n]), return_lse=True, max_prefix=n, max_own=own)
    assert bool(clean[0].isfinite().all() and clean[1].isfinite().all())
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    for tok in ([0, 6, 7, 16, 17, 40, 5003, 19999] if where == "prefix" else [n]):
        o, lse = prefix_decode(q, plant(kp, bt, zero, zero + tok, page, what), vp, bt, lens, ints([0, R]), ints([n]),
                               return_lse=True, max_prefix=n, max_own=own)
        hit = poisoned(o, lse)
        assert bool(hit.all() if where == "prefix" else hit[0].all() and not hit[1:].any()), tok
        if where == "own":
            assert torch.equal(o[1:], clean[0][1:]) and torch.equal(lse[1:], clean[1][1:])
