"""Rotary positions and copies inside the paged cache against plain 64-bit
forms.

Tolerances: a rotated value y is a sum of two products of magnitude at most
m max|x| (m: the largest table entry), each rounded to fp32 (2^-24) or fused,
and is rounded once to the data's type, whose unit roundoff is u = 2^-8 (bf16),
2^-11 (fp16), 0 (fp32, counted already).  So each element holds
|error| <= u |y| + 8 * 2^-24 m max|x| + 2^-25, the last for fp16's subnormals.
Copies are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def _near(got, want, x, dtype, m=1.0):
    """Whether each element of got is as near to the 64-bit want as one rounding allows (x: what was turned)."""
    tol = UNIT[dtype] * want.abs() + 8 * 2.0 ** -24 * m * float(x.abs().max()) + 2.0 ** -25
    return bool(((got.detach().double() - want).abs() <= tol).all())


def _turn(x, cos, sin, layout, sign=1.0):
    """x [..., D] in 64 bits, cos / sin [..., rot / 2]."""
    x, c, s = x.double(), cos.double(), sign * sin.double()
    h = c.shape[-1]
    y = x.clone()
    if layout == "half":
        a, b = x[..., :h], x[..., h:2 * h]
        y[..., :h], y[..., h:2 * h] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = a * c - b * s, b * c + a * s
    return y


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,storage", [
    (1, 1, 1, 1, 64, 64, "bshd"),       # one token, one head
    (2, 77, 8, 2, 128, 128, "bshd"),    # grouped heads, a ragged length
    (3, 33, 5, 1, 96, 48, "bhsd"),      # part of the head, contiguous heads
    (2, 129, 7, 7, 64, 20, "bshd"),     # a rotated width no vector divides
    (1, 300, 32, 8, 128, 64, "slice"),  # slices of a stacked projection
    (2, 40, 3, 3, 72, 72, "odd"),       # storage no vector load can take
])
def test_apply_rotary_and_gradient(B, S, Hq, Hkv, D, rot, storage, dtype, layout):
    from fastest_flash_attention_b200 import apply_rotary, rotary_tables
    g = _gen(B * S + D)
    if storage == "bhsd":
        q, k = (torch.randn(B, h, S, D, generator=g, device="cuda").to(dtype) for h in (Hq, Hkv))
    elif storage == "bshd":
        q, k = (torch.randn(B, S, h, D, generator=g, device="cuda").to(dtype).transpose(1, 2) for h in (Hq, Hkv))
    elif storage == "slice":
        x = torch.randn(B, S, (Hq + Hkv) * D, generator=g, device="cuda").to(dtype)
        q = x[..., :Hq * D].view(B, S, Hq, D).transpose(1, 2)
        k = x[..., Hq * D:].view(B, S, Hkv, D).transpose(1, 2)
    else:
        q, k = (torch.randn(B, S, h, D + 3, generator=g, device="cuda").to(dtype)[..., 1:D + 1].transpose(1, 2)
                for h in (Hq, Hkv))
    cos, sin = rotary_tables(rot, 1000)
    pos = torch.randint(0, 1000, (B, S), generator=g, device="cuda")
    qr, kr = q.detach().requires_grad_(), k.detach().requires_grad_()
    qo, ko = apply_rotary(qr, kr, cos, sin, pos, layout=layout)
    c, s = cos[pos][:, None], sin[pos][:, None]
    dq, dk = torch.randn_like(qo), torch.randn_like(ko)
    gq, gk = torch.autograd.grad((qo, ko), (qr, kr), (dq, dk))
    for got, x, sign in ((qo, q, 1.0), (ko, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        assert got.shape == x.shape and got.dtype == dtype
        assert _near(got, _turn(x, c, s, layout, sign), x, dtype)
    assert torch.equal(qo[..., rot:], q[..., rot:]) and torch.equal(gk[..., rot:], dk[..., rot:])
    # int32 positions, one row for all, no k: the same values
    q1, none = apply_rotary(q, None, cos, sin, pos[0].to(torch.int32), layout=layout)
    assert none is None and torch.equal(q1[0], qo[0])


def test_rotary_gradient_against_differences():
    """fp32, central differences of a random projection of the output: the
    rotation is linear, so the difference quotient is exact up to the rounding
    of two fp32 outputs (2^-23 each, of values below 2^3, over a step of 2)."""
    from fastest_flash_attention_b200 import apply_rotary, rotary_tables
    g = _gen(7)
    q = torch.randn(1, 2, 3, 16, generator=g, device="cuda")
    w = torch.randn(1, 2, 3, 16, generator=g, device="cuda").double()
    cos, sin = rotary_tables(8, 64, scaling="yarn", factor=4.0, original_max_len=16)
    x = q.clone().requires_grad_()
    out, _ = apply_rotary(x, None, cos, sin, 5, layout="interleaved")
    (grad,) = torch.autograd.grad(out, x, w.float())
    for i in range(q.numel()):
        e = torch.zeros_like(q).view(-1)
        e[i] = 1.0
        up, _ = apply_rotary(q + e.view_as(q), None, cos, sin, 5, layout="interleaved")
        dn, _ = apply_rotary(q - e.view_as(q), None, cos, sin, 5, layout="interleaved")
        diff = float(((up.double() - dn.double()) / 2 * w).sum())
        assert abs(diff - float(grad.view(-1)[i])) <= 96 * 2.0 ** -23 * 8 * 4


def test_rotary_only_one_gradient_and_empty():
    from fastest_flash_attention_b200 import apply_rotary, rotary_tables
    cos, sin = rotary_tables(32, 16)
    q = torch.randn(2, 3, 9, 32, device="cuda", requires_grad=True)
    k = torch.randn(2, 1, 9, 32, device="cuda", requires_grad=True)
    qo, ko = apply_rotary(q, k, cos, sin, 3)
    (gk,) = torch.autograd.grad(ko.sum(), k)
    want = _turn(torch.ones_like(k), cos[3:12][None, None], sin[3:12][None, None], "half", -1.0)
    assert _near(gk, want, torch.ones(1), torch.float32)
    e, _ = apply_rotary(torch.zeros(2, 3, 0, 32, device="cuda"), None, cos, sin, 16)
    assert e.shape == (2, 3, 0, 32)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,T,Hq,Hkv,D,rot,page", [
    (torch.bfloat16, 1, 32, 8, 128, 128, 16),
    (torch.float16, 64, 20, 5, 64, 32, 24),
    (torch.bfloat16, 333, 7, 1, 96, 20, 64),
    (torch.float32, 17, 4, 2, 40, 40, 5),
])
def test_rotary_append(dtype, T, Hq, Hkv, D, rot, page, layout):
    from fastest_flash_attention_b200 import rotary_append, rotary_tables
    g = _gen(T)
    x = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(dtype)
    q, k, v = x[:, :Hq * D].view(T, Hq, D), x[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D), \
        x[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    P = 2 * T // page + 2
    kp, vp = (torch.randn(P, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    kw, vw = kp.double(), vp.double()
    cos, sin = rotary_tables(rot, 5000)
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda")
    slots = torch.randperm(P * page, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 1:
        slots[0] = -1  # a padding token writes nothing
    qo = rotary_append(q, k, v, cos, sin, pos, slots, kp, vp, layout=layout)
    c, s = cos[pos][:, None], sin[pos][:, None]
    live = slots >= 0
    sl = slots[live].long()
    kw[sl // page, :, sl % page] = _turn(k, c, s, layout)[live]
    vw[sl // page, :, sl % page] = v.double()[live]
    assert _near(qo, _turn(q, c, s, layout), q, dtype) and _near(kp, kw, k, dtype)
    assert torch.equal(vp.double(), vw)


@pytest.mark.parametrize("dtype,P,Hkv,page,D,n", [
    (torch.bfloat16, 40, 8, 64, 128, 16),
    (torch.float16, 9, 3, 5, 24, 4),      # pages no 16-byte multiple of a tile
    (torch.float32, 7, 1, 16, 64, 3),
    (torch.float16, 6, 1, 3, 3, 2),       # 18 bytes a page: the narrow copy
    (torch.uint8, 8, 2, 16, 64, 4),       # any type
])
def test_copy_pages(dtype, P, Hkv, page, D, n):
    from fastest_flash_attention_b200 import copy_pages
    g = _gen(P)
    kp, vp = ((torch.randn(P, Hkv, page, D, generator=g, device="cuda") * 9).to(dtype) for _ in range(2))
    order = torch.randperm(P, generator=g, device="cuda")
    src, dst = order[:n], order[n:2 * n]
    kw, vw = kp.clone(), vp.clone()
    kw[dst], vw[dst] = kp[src], vp[src]
    k2 = kp.clone()
    copy_pages(kp, vp, src.to(torch.int32), dst)
    assert torch.equal(kp, kw) and torch.equal(vp, vw)
    copy_pages(k2, None, src.tolist(), dst.tolist())  # one pool, ids on the host
    assert torch.equal(k2, kw)
    copy_pages(kp, vp, [], [])
    assert torch.equal(kp, kw)


@pytest.mark.parametrize("dtype,P,Hkv,page,D,n", [
    (torch.bfloat16, 64, 8, 16, 128, 400),
    (torch.float16, 20, 5, 24, 64, 1),
    (torch.bfloat16, 33, 3, 5, 72, 80),
    (torch.float16, 9, 2, 7, 5, 20),      # 10-byte rows: the narrow copy
    (torch.float32, 16, 0, 16, 96, 64),   # a latent cache: [P, page, D]
])
def test_move_tokens(dtype, P, Hkv, page, D, n):
    from fastest_flash_attention_b200 import move_tokens
    g = _gen(n)
    shape = (P, Hkv, page, D) if Hkv else (P, page, D)
    kp, vp = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    order = torch.randperm(P * page, generator=g, device="cuda")
    src, dst = order[:n].to(torch.int32), order[n:2 * n].to(torch.int32)
    want = []
    for pool in (kp, vp):
        w = pool.clone().view(P, max(Hkv, 1), page, D)
        s, d = src.long(), dst.long()
        w[d // page, :, d % page] = w[s // page, :, s % page]
        want.append(w.view(shape))
    move_tokens(kp, vp, src, dst)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_ids_outside_the_pool_and_tables_are_reported():
    from fastest_flash_attention_b200 import apply_rotary, copy_pages, move_tokens, rotary_tables
    kp = torch.randn(4, 2, 8, 16, device="cuda")
    keep = kp.clone()
    bad = torch.tensor([4], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="outside the pool"):
        copy_pages(kp, None, bad, torch.tensor([1], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="outside the pool"):
        move_tokens(kp, None, torch.tensor([0], dtype=torch.int32, device="cuda"), bad * 8)
    assert torch.equal(kp, keep)
    cos, sin = rotary_tables(16, 10)
    with pytest.raises(RuntimeError, match="outside the cos / sin tables"):
        apply_rotary(kp, None, cos, sin, torch.full((8,), 10, dtype=torch.int32, device="cuda"))


def test_cache_fork_trim_compact():
    """Forked, trimmed and compacted sequences hold the tokens they should, and
    every page comes back in the end."""
    from fastest_flash_attention_b200 import PagedKVCache
    g = _gen(1)
    H, D, ps = 2, 64, 16
    c = PagedKVCache(max_pages=64, page_size=ps, num_heads=H, head_dim=D, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.randn(H, 133, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    c.append_tokens(0, k, v)
    free = c.num_free_pages
    c.fork_sequences([(0, 1), (0, 2)])
    assert free - c.num_free_pages == 2  # only the two last pages
    k1, v1 = (torch.randn(H, 9, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    c.append_tokens(1, k1, v1)
    assert torch.equal(c.get_kv(0)[0], k) and torch.equal(c.get_kv(2)[1], v)
    assert torch.equal(c.get_kv(1)[0], torch.cat([k, k1], 1))
    assert c.trim_sequence(2, 40, 4) == 0  # shared with the other two: nothing comes free yet
    with pytest.raises(RuntimeError, match="were freed"):
        c.get_kv(2)
    assert c.compact_sequences([1, 0], 40, 4) == (142 - 44) + (133 - 44)
    assert torch.equal(c.get_kv(0)[0], torch.cat([k[:, :4], k[:, -40:]], 1))
    assert torch.equal(c.get_kv(1)[1], torch.cat([v[:, :4], v[:, -31:], v1], 1))
    assert c.position(0) == 133 and c.position(1) == 142
    c.append_tokens(0, k1, v1)
    assert c.position(0) == 142 and torch.equal(c.get_kv(0)[0][:, -9:], k1)
    for s in (0, 1, 2):
        c.free_sequence(s)
    assert sorted(c.free_pages) == list(range(64)) and not c._more_owners
