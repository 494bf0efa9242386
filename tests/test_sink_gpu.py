"""Attention with a sliding window and the first tokens kept visible: forward
and gradients against 64-bit automatic differentiation of the formula.

Tolerances, derived beforehand, relative to each result's own root mean square
(the sums below are over independent roundings, so norms add in quadrature and
4x is allowed for the largest element's share):
  16-bit types, unit roundoff u (2^-8 bf16, 2^-11 fp16): O, dQ, dK, dV are
  rounded once (rms u / sqrt(3) at most) and their products' P or dS operand
  once before (the same).  The norm of the error is held to 2 u of the norm of
  the result, each LSE to 2^-10 (fp32 sums of exact products, scores below 40).
  fp32: products and sums of up to 600 terms in fp32 at 2^-24 each, through
  exp of scores below 40: norms within 1e-5 (O, LSE) and 1e-4 (gradients), the
  bounds the fp32 path holds everywhere.
Where a row's softmax sits on one key, dS = P (dP - Delta) cancels and the
gradients lose what Delta = rowsum(dO O) does: the backward takes the rounded O,
so Delta is off by at most e = (u + 64 * 2^-24) rowsum|dO O| (u = 0 for fp32; 64:
the fp32 sums of D products on both sides).  That moves dQ by at most
scale e P |K| and dK by scale P^T (e |Q|), element by element, which is allowed
on top."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _visible(Sq, Skv, window, sinks, causal, off):
    i = torch.arange(Sq, device="cuda")[:, None] + off
    j = torch.arange(Skv, device="cuda")[None, :]
    keep = (j > i - window) | (j < sinks)
    return keep & (j <= i) if causal else keep


def _exact(q, k, v, do, keep, softcap, scale):
    """o, lse, dq, dk, dv in 64 bits, and how far Delta's rounding may move dq
    and dk; rows that see nothing give 0 and -inf."""
    u = U.get(q.dtype, 0.0)
    q, k, v = (t.detach().double().requires_grad_() for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    kk, vv = (t.repeat_interleave(G, 1) for t in (k, v))
    s = q @ kk.transpose(-1, -2) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    seen = keep.any(-1)
    s = torch.where(keep, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, torch.exp(s - torch.where(seen, lse, 0.0)[..., None]), 0.0)
    o = p @ vv
    grads = torch.autograd.grad(o, (q, k, v), do.double())
    with torch.no_grad():
        e = (u + 64 * 2.0 ** -24) * (do.double() * o).abs().sum(-1, keepdim=True)
        mq = scale * e * (p @ kk.abs())
        mk = scale * (p.transpose(-1, -2) @ (e * q.abs()))
        mk = mk.view(k.shape[0], k.shape[1], G, *k.shape[2:]).sum(2)
    return (o, lse) + grads + (dict(dq=mq, dk=mk),)


def _near(got, want, dtype, name, more=None):
    got, want = got.detach().double(), want.detach()
    more = (more or {}).get(name, torch.zeros((), dtype=torch.float64, device="cuda"))
    tol = 2 * U[dtype] if dtype in U else (1e-5 if name == "o" else 1e-4)
    assert bool(torch.isfinite(got).all()), name
    norm = float(want.norm())
    err = float((got - want).norm())
    assert err <= tol * norm + float(more.norm()), (name, err / max(norm, 1e-300), tol)
    rms = norm / math.sqrt(max(want.numel(), 1))
    assert bool(((got - want).abs() <= 16 * tol * torch.clamp(want.abs(), min=rms) + more).all()), name


def _tensors(B, Hq, Hkv, Sq, Skv, D, Dv, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(h, s, d):  # [B, S, H, D] storage, as the projections leave it
        return torch.randn(B, s, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
    return t(Hq, Sq, D), t(Hkv, Skv, D), t(Hkv, Skv, Dv), t(Hq, Sq, Dv)


CASES = [
    # B, Hq, Hkv, Sq, Skv, D, Dv, window, sinks, causal, softcap
    (1, 1, 1, 1, 1, 64, 64, 1, 1, True, None),            # one token
    (2, 4, 2, 77, 77, 128, 128, 32, 3, True, None),       # under one tile
    (1, 4, 1, 777, 777, 128, 128, 128, 4, True, None),    # ragged, window of a tile
    (1, 2, 2, 1300, 1300, 64, 64, 200, 17, True, 30.0),   # sinks inside a tile, softcap
    (1, 3, 3, 1025, 1025, 128, 128, 1, 1, True, None),    # each query sees itself and the first key
    (2, 6, 2, 900, 900, 64, 64, 100, 130, True, None),    # sinks past one key tile
    (1, 2, 1, 640, 640, 128, 128, 65, 700, True, None),   # every key a sink: plain causal
    (1, 2, 1, 500, 500, 128, 128, 4000, 4, True, None),   # a window that hides nothing
    (1, 4, 2, 600, 600, 192, 128, 150, 5, True, None),    # qk 192, v 128
    (1, 2, 2, 513, 513, 96, 96, 64, 9, True, 20.0),       # head dims below the tile's
    (2, 4, 2, 300, 300, 40, 24, 50, 3, True, None),       # ... of q / k and v apart
    (1, 2, 1, 777, 777, 136, 72, 128, 4, True, None),     # ... on the widest tile
    (1, 2, 2, 200, 200, 20, 20, 30, 3, True, None),       # no multiple of 8: padded copies
    (1, 2, 1, 400, 1100, 64, 64, 90, 6, True, None),      # more keys than queries (offset 0)
    (1, 2, 1, 1100, 400, 128, 128, 90, 6, False, None),   # windows past the last key: sinks alone
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,D,Dv,window,sinks,causal,softcap", CASES)
def test_forward_and_gradients(B, Hq, Hkv, Sq, Skv, D, Dv, window, sinks, causal, softcap, dtype):
    from fastest_flash_attention_b200 import fastest_flash_attn_forward, fastest_flash_attn_func
    q, k, v, do = _tensors(B, Hq, Hkv, Sq, Skv, D, Dv, dtype, Sq + D)
    keep = _visible(Sq, Skv, window, sinks, causal, 0)
    want = _exact(q, k, v, do, keep, softcap, 1 / math.sqrt(D))
    o, lse = fastest_flash_attn_forward(q, k, v, causal=causal, sliding_window=window, sink_tokens=sinks,
                                        softcap=softcap, return_lse=True)
    assert o.dtype == dtype and lse.shape == (B, Hq, Sq, 1)
    _near(o, want[0], dtype, "o")
    assert float((lse[..., 0].double() - want[1]).abs().max()) <= (2.0 ** -10 if dtype in U else 1e-5 * 40)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = fastest_flash_attn_func(q, k, v, causal=causal, sliding_window=window, sink_tokens=sinks, softcap=softcap)
    assert torch.equal(out, o)
    grads = torch.autograd.grad(out, (q, k, v), do)
    for name, got, ref in zip(("dq", "dk", "dv"), grads, want[2:]):
        _near(got, ref, dtype, name, want[5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off,window,sinks", [(-40, 16, 3), (-300, 50, 0), (300, 64, 5), (1000, 10, 200)])
def test_offsets_and_rows_that_see_nothing(off, window, sinks, dtype):
    """Queries before the first key see nothing (0, LSE -inf, no gradient);
    queries past the last key's window see the sinks alone."""
    from fastest_flash_attention_b200.attention import flash_bwd, flash_fwd
    q, k, v, do = _tensors(1, 4, 2, 333, 290, 64, 64, dtype, 5)
    keep = _visible(333, 290, window, sinks, True, off)
    want = _exact(q, k, v, do, keep, None, 0.125)
    o, lse = flash_fwd(q, k, v, scale=0.125, causal=True, q_offset=off, window=window, sink=sinks)
    blind = ~keep.any(-1)
    assert bool((lse[..., blind] == -math.inf).all()) and bool((o[:, :, blind] == 0).all())
    seen = ~blind
    if bool(seen.any()):
        assert float((lse[..., seen].double() - want[1][..., seen]).abs().max()) <= 2.0 ** -10
    _near(o, want[0], dtype, "o")
    grads = flash_bwd(do, q, k, v, o, lse, scale=0.125, causal=True, q_offset=off, window=window, sink=sinks)
    for name, got, ref in zip(("dq", "dk", "dv"), grads, want[2:]):
        _near(got, ref, dtype, name, want[5])


@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (192, 128)])
def test_long_sequence_backward_is_bit_identical(D, Dv):
    """Many query shares of the sink tile: the same bits twice, and near the formula."""
    from fastest_flash_attention_b200 import fastest_flash_attn_func
    q, k, v, do = _tensors(1, 4, 2, 5000, 5000, D, Dv, torch.bfloat16, 9)
    runs = []
    for _ in range(2):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        out = fastest_flash_attn_func(*x, causal=True, sliding_window=130, sink_tokens=4)
        runs.append((out,) + torch.autograd.grad(out, x, do))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    want = _exact(q, k, v, do, _visible(5000, 5000, 130, 4, True, 0), None, 1 / math.sqrt(D))
    for name, got, ref in zip(("o", "dq", "dk", "dv"), runs[0], (want[0],) + want[2:5]):
        _near(got, ref, torch.bfloat16, name, want[5])


def test_gradient_against_differences():
    """fp32, central differences along random directions: the difference
    quotient over a step h = 2^-6 is off by the third derivative (at most
    h^2 / 6 of the second-order scale, below 2^-13 of the directional
    derivative's own scale here) and by rounding 2^-22 |f| / h."""
    from fastest_flash_attention_b200 import fastest_flash_attn_func
    q, k, v, do = _tensors(1, 2, 1, 150, 150, 64, 64, torch.float32, 3)
    kw = dict(causal=True, sliding_window=20, sink_tokens=3, softcap=15.0)

    def f(a, b, c):
        return float((fastest_flash_attn_func(a, b, c, **kw).double() * do.double()).sum())
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(fastest_flash_attn_func(*x, **kw), x, do)
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(3):
        for _ in range(3):
            d = torch.randn(x[i].shape, generator=g, device="cuda")
            d = d / d.norm()
            h = 2.0 ** -6
            up, dn = [t.detach() for t in x], [t.detach() for t in x]
            up[i], dn[i] = up[i] + h * d, dn[i] - h * d
            slope = (f(*up) - f(*dn)) / (2 * h)
            scale = float(grads[i].norm())
            assert abs(slope - float((grads[i].double() * d.double()).sum())) <= 2.0 ** -9 * scale


def test_no_sinks_and_no_window_change_nothing():
    from fastest_flash_attention_b200 import AttentionConfig, fastest_flash_attn_forward
    q, k, v, _ = _tensors(1, 4, 2, 700, 700, 128, 128, torch.bfloat16, 1)
    a, _ = fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=100)
    b, _ = fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=100, sink_tokens=0)
    assert torch.equal(a, b)
    a, _ = fastest_flash_attn_forward(q, k, v, causal=True)
    b, _ = fastest_flash_attn_forward(q, k, v, causal=True, sink_tokens=7)
    assert torch.equal(a, b)
    a, _ = fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=100, sink_tokens=7)
    b, _ = fastest_flash_attn_forward(q, k, v, AttentionConfig(causal=True, sliding_window=100, sink_tokens=7))
    assert torch.equal(a, b)


def test_windows_and_sinks_past_any_length():
    from fastest_flash_attention_b200 import fastest_flash_attn_forward, fastest_flash_attn_func
    q, k, v, do = _tensors(1, 4, 2, 300, 300, 64, 64, torch.float16, 2)
    want, _ = fastest_flash_attn_forward(q, k, v, causal=True)
    for kw in (dict(sliding_window=2 ** 40), dict(sliding_window=2 ** 31, sink_tokens=3),
               dict(sliding_window=1, sink_tokens=2 ** 40)):
        o, _ = fastest_flash_attn_forward(q, k, v, causal=True, **kw)
        assert torch.equal(o, want)
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        g = torch.autograd.grad(fastest_flash_attn_func(*x, causal=True, **kw), x, do)
        ref = torch.autograd.grad(fastest_flash_attn_func(*x, causal=True), x, do)
        for name, a, b in zip(("dq", "dk", "dv"), g, ref):  # both are one rounding of nearly the same sums
            _near(a, b.double(), torch.float16, name)


def test_many_sink_tiles():
    """Sinks over dozens of key tiles: each tile's queries are shared by few CTAs."""
    from fastest_flash_attention_b200 import fastest_flash_attn_func
    q, k, v, do = _tensors(1, 2, 1, 6000, 6000, 64, 64, torch.bfloat16, 6)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    out = fastest_flash_attn_func(*x, causal=True, sliding_window=60, sink_tokens=4500)
    grads = torch.autograd.grad(out, x, do)
    want = _exact(q, k, v, do, _visible(6000, 6000, 60, 4500, True, 0), None, 0.125)
    for name, got, ref in zip(("o", "dq", "dk", "dv"), (out,) + grads, (want[0],) + want[2:5]):
        _near(got, ref, torch.bfloat16, name, want[5])


def test_three_dimensional_tensors():
    from fastest_flash_attention_b200 import fastest_flash_attn_forward, fastest_flash_attn_func
    q, k, v, do = (t[:, 0] for t in _tensors(2, 1, 1, 200, 200, 64, 64, torch.bfloat16, 8))
    kw = dict(causal=True, sliding_window=30, sink_tokens=4)
    o, lse = fastest_flash_attn_forward(q, k, v, return_lse=True, **kw)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    out = fastest_flash_attn_func(*x, **kw)
    assert out.shape == q.shape and torch.equal(out, o) and lse.shape == (2, 200, 1)
    got = torch.autograd.grad(out, x, do)
    x = [t.detach().unsqueeze(1).requires_grad_() for t in (q, k, v)]
    ref = torch.autograd.grad(fastest_flash_attn_func(*x, **kw), x, do.unsqueeze(1))
    assert all(torch.equal(a, b[:, 0]) for a, b in zip(got, ref))


def test_refusals():
    from fastest_flash_attention_b200 import fastest_flash_attn_backward, fastest_flash_attn_forward
    q, k, v, do = _tensors(1, 2, 2, 64, 64, 64, 64, torch.bfloat16, 1)
    mask = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    for kw in (dict(sink_tokens=-1), dict(sliding_window=8, sink_tokens=-1),
               dict(sliding_window=8, sink_tokens=2, block_mask=mask, block_size=64)):
        with pytest.raises(ValueError):
            fastest_flash_attn_forward(q, k, v, causal=True, **kw)
    o, lse = fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=8, sink_tokens=2, return_lse=True)
    with pytest.raises(ValueError):
        fastest_flash_attn_backward(do, q, k, v, o, lse, causal=True, sliding_window=8, sink_tokens=2,
                                    block_mask=mask)


def test_modules_take_sinks():
    from fastest_flash_attention_b200 import FastestFlashGQA, FastestFlashMHA, fastest_flash_attn_forward
    torch.manual_seed(0)
    m = FastestFlashGQA(256, 4, 2, causal=True, sliding_window=30, sink_tokens=4).cuda().to(torch.bfloat16)
    x = torch.randn(2, 200, 256, device="cuda", dtype=torch.bfloat16)
    q = m.q_proj(x).view(2, 200, 4, 64).transpose(1, 2)
    k, v = (p(x).view(2, 200, 2, 64).transpose(1, 2) for p in (m.k_proj, m.v_proj))
    o, _ = fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=30, sink_tokens=4)
    want = m.o_proj(o.transpose(1, 2).reshape(2, 200, -1))
    assert torch.equal(m.eval()(x), want) and torch.equal(m.train()(x), want)
    plain = FastestFlashMHA(256, 4, causal=True, sliding_window=30).cuda().to(torch.bfloat16).eval()
    sinks = FastestFlashMHA(256, 4, causal=True, sliding_window=30, sink_tokens=4).cuda().to(torch.bfloat16).eval()
    sinks.load_state_dict(plain.state_dict())
    # token 30 is the first whose window has left token 0
    assert torch.equal(sinks(x)[:, :30], plain(x)[:, :30]) and not torch.equal(sinks(x)[:, 30:], plain(x)[:, 30:])
