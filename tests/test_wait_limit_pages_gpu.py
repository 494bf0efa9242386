"""Bounded in-kernel waits of the query rows over pages: with a limit of 1 ns half of the
CTAs' first wait of the products and the others' last wait for O run out unless they are
complete at once.  The kernel records its site, every role stops waiting, copies and
products in flight finish (draining waits keep a floor of seconds whatever the limit) and
it returns; a launch behind it joins whatever it left.  The host sees the error, the
context stays usable, and the next call with the default limit gives the same bits as the
one before.  No fault, trap or hang is involved."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(rows, n, page, Hkv, D, dtype, shared=0):
    g = torch.Generator(device="cuda").manual_seed(n + D)
    per = -(-n // page)
    bt = torch.randperm(rows * per, generator=g, device="cuda").view(rows, per).int()
    bt[:, :shared // page] = bt[0, :shared // page]
    kp, vp = (torch.randn(rows * per, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    return kp, vp, bt, g


def expires(call):
    from fastest_flash_attention_b200 import _lib
    lib, dev = _lib.load(), torch.device("cuda", 0)
    before = call()
    torch.cuda.synchronize()
    _lib.check_device_errors(dev)
    for _ in range(3):
        lib.ffa_set_wait_limit_ns(1)
        try:
            with pytest.raises(RuntimeError, match="FFA_ERR_DEVICE_TIMEOUT") as e:
                call()
                torch.cuda.synchronize()
                _lib.check_device_errors(dev)
            assert 0x501 <= int(str(e.value).split("site 0x")[1].split()[0], 16) <= 0x506  # (not the drain's)
        finally:
            lib.ffa_set_wait_limit_ns(0)  # back to the default
        after = call()
        torch.cuda.synchronize()
        _lib.check_device_errors(dev)
        assert all(torch.equal(a, b) for a, b in zip(before, after))


# tokens, new, Hq, Hkv, D, dtype: two query tiles; one; 32 rows, split and joined; D 64; more CTAs than fit at once
@pytest.mark.parametrize("R,n,new,Hq,Hkv,D,dtype", [
    (1, 2000, 700, 8, 2, 128, torch.bfloat16), (2, 900, 100, 2, 2, 128, torch.float16),
    (1, 6000, 3, 32, 8, 128, torch.bfloat16), (3, 700, 300, 4, 4, 64, torch.float16),
    (40, 600, 200, 8, 8, 64, torch.bfloat16), (64, 300, 150, 8, 8, 128, torch.bfloat16)])
def test_prefill(R, n, new, Hq, Hkv, D, dtype):
    from fastest_flash_attention_b200 import paged_prefill
    kp, vp, bt, g = pool(R, n, 16, Hkv, D, dtype)
    q = torch.randn(R * new, Hq, D, generator=g, device="cuda").to(dtype)
    lens, starts = ints([n] * R), ints([i * new for i in range(R + 1)])
    expires(lambda: paged_prefill(q, kp, vp, bt, lens, starts, return_lse=True))


# two launches (own tokens joined by the second), and three
@pytest.mark.parametrize("R,prefix,Hq,Hkv,D,dtype", [(64, 8192, 32, 8, 128, torch.bfloat16),
                                                     (40, 20000, 8, 4, 64, torch.float16)])
def test_prefix(R, prefix, Hq, Hkv, D, dtype):
    from fastest_flash_attention_b200 import prefix_decode
    kp, vp, bt, g = pool(R, prefix + 32, 16, Hkv, D, dtype, shared=prefix)
    q = torch.randn(R, Hq, D, generator=g, device="cuda").to(dtype)
    lens, starts, prefixes = ints([prefix + 1 + i % 32 for i in range(R)]), ints([0, R]), ints([prefix])
    expires(lambda: prefix_decode(q, kp, vp, bt, lens, starts, prefixes, return_lse=True, max_prefix=prefix, max_own=32))
