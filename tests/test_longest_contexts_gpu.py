"""Contexts of nearly 2^31 tokens, the longest that the entry points take (one page,
again and again): positions, shares and their number are right up there.

All scores are 0 and V is one row, so O is that row and the LSE ln n.  P is within
2^-18 of 1 and rounds to it; the row sum of n / 64 shares rounds to whole numbers: O
is off by its own rounding and, through the sum, by 2^-17, the LSE by 2^-10 (its fp32
rounding and that of the scores, as in test_paged_prefill_gpu.py).  O's sum over a
share grows to n / 64 = 2^25 products V, and the tensor core cuts each product off at
the last of the some 25 bits that it keeps of the sum: what is kept of V is between
its leading bit, which stands 2^25 below the sum at most, and V.  So O is exact to the
above where V is a power of two, and elsewhere between that leading bit and V."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, WIDTH = 65536, 32767


def make(rows):
    kp = torch.randn(1, 1, PAGE, 8, device="cuda").half()
    vp = torch.arange(1, 9, device="cuda").half().expand(1, 1, PAGE, 8).contiguous()
    return kp, vp, torch.zeros(rows, WIDTH, dtype=torch.int32, device="cuda")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(o, lse, vp, lens):
    want = vp[0, 0, 0].double()
    lead, eps = 2.0 ** want.log2().floor(), 2.0 ** -11 + 2.0 ** -17
    assert bool((o.double() >= lead * (1 - eps)).all()) and bool((o.double() <= want * (1 + eps)).all())
    assert float((lse.double() - torch.tensor(lens, device="cuda").double().log()[:, None]).abs().max()) <= 2.0 ** -10


def test_prefill():
    from fastest_flash_attention_b200 import paged_prefill
    n = PAGE * WIDTH
    kp, vp, bt = make(1)
    q = torch.zeros(2, 2, 8, device="cuda", dtype=torch.float16)
    o, lse = paged_prefill(q, kp, vp, bt, ints([n]), ints([0, 2]), return_lse=True)
    check(o, lse, vp, [n - 1, n])


def test_prefix():
    from fastest_flash_attention_b200 import prefix_decode
    n = PAGE * (WIDTH - 1)
    kp, vp, bt = make(3)
    lens = [n + 5, n, n + PAGE]
    q = torch.zeros(3, 1, 8, device="cuda", dtype=torch.float16)
    o, lse = prefix_decode(q, kp, vp, bt, ints(lens), ints([0, 3]), ints([n]), return_lse=True, max_own=PAGE)
    check(o, lse, vp, lens)
    assert math.isfinite(float(lse.sum()))
