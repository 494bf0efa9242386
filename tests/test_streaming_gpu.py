"""The streaming module and its decoder: training gradients against 64-bit
automatic differentiation, and decoding (with forks, freed pages and
compaction) against the module run over the whole sequence.

Tolerances, derived beforehand: q, k, v, the attention's output and the result
are each rounded to bf16 once more in one of the two runs than in the other
or in the 64-bit form (u = 2^-8 each, relative to the norm: sqrt(3) smaller on
average); six such roundings in quadrature, and twice that allowed:
2 * sqrt(6) * u / sqrt(3) < 3 u of the result's norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def _module(**kw):
    from fastest_flash_attention_b200 import FastestFlashStreamingGQA
    torch.manual_seed(0)
    args = dict(sliding_window=70, sink_tokens=5, max_len=1024)
    args.update(kw)
    return FastestFlashStreamingGQA(256, 4, 2, **args).cuda().to(torch.bfloat16)


def _near(got, want, n=3.0):
    got, want = got.detach().double(), want.detach().double()
    assert float((got - want).norm()) <= n * U * float(want.norm())


def _exact(m, x):
    """The module in 64 bits, differentiable, from its own parameters and tables."""
    B, S, _ = x.shape
    H, Hkv, D = m.num_heads, m.num_kv_heads, m.head_dim
    P = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    cos, sin = (t[:S].double() for t in m.tables(x.device))
    h = cos.shape[1]

    def heads(name, n):
        return (x @ P[name + "_proj.weight"].T).view(B, S, n, D).transpose(1, 2)

    def turn(t):
        if m.rotary_layout == "half":
            a, b = t[..., :h], t[..., h:2 * h]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, t[..., 2 * h:]], -1)
        a, b = t[..., 0:2 * h:2], t[..., 1:2 * h:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), t[..., 2 * h:]], -1)
    q, k, v = turn(heads("q", H)), turn(heads("k", Hkv)), heads("v", Hkv)
    k, v = (t.repeat_interleave(H // Hkv, 1) for t in (k, v))
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None, :]
    seen = (j <= i) & ((j > i - m.sliding_window) | (j < m.sink_tokens))
    p = torch.softmax((q @ k.transpose(-1, -2) * m.scale).masked_fill(~seen, -math.inf), -1)
    return (p @ v).transpose(1, 2).reshape(B, S, -1) @ P["o_proj.weight"].T, P


@pytest.mark.parametrize("kw", [dict(), dict(rotary_layout="interleaved", rotary_dim=32),
                                dict(rotary_scaling=dict(scaling="yarn", factor=4.0, original_max_len=256))])
def test_training_step(kw):
    m = _module(**kw).train()
    x = torch.randn(2, 300, 256, device="cuda", dtype=torch.bfloat16)
    out = m(x)
    want, P = _exact(m, x.double())
    _near(out, want)
    g = torch.randn_like(out)
    names, params = zip(*m.named_parameters())
    got = torch.autograd.grad(out, params, g)
    ref = torch.autograd.grad(want, [P[n] for n in names], g.double())
    for n, a, b in zip(names, got, ref):
        _near(a, b, 4.0)  # one more chain of roundings behind the attention
    assert torch.equal(m.eval()(x), out)


def test_decoding_matches_the_whole_sequence():
    from fastest_flash_attention_b200 import StreamingDecoder
    m = _module().eval()
    dec = StreamingDecoder(m, max_pages=40, page_size=16)
    x = torch.randn(2, 330, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        whole = m(x)
    first = dec.prefill(x[:, :250], [0, 1])
    _near(first, whole[:, :250])
    held = [p for p in dec.cache.sequences[0]["page_table"] if p >= 0]
    assert len(held) <= 70 // 16 + 2 + 1  # window and first tokens alone
    for t in range(250, 280):
        _near(dec.step(x[:, t:t + 1], [0, 1]), whole[:, t:t + 1])
    dec.fork([(0, 7)])
    other = torch.randn(1, 1, 256, device="cuda", dtype=torch.bfloat16)
    dec.step(other, [7])  # the fork goes its own way
    assert dec.compact([0, 1]) > 0
    for t in range(280, 330):
        _near(dec.step(x[:, t:t + 1], [0, 1]), whole[:, t:t + 1])
    assert dec.cache.position(7) == 281 and dec.cache.position(0) == 330
    last = torch.randn(1, 1, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        forked = m(torch.cat([x[:1, :280], other, last], 1))
    _near(dec.step(last, [7]), forked[:, -1:])
    for s in (0, 1, 7):
        dec.free(s)
    assert dec.cache.num_free_pages == 40


def test_refusals():
    from fastest_flash_attention_b200 import FastestFlashStreamingGQA, StreamingDecoder
    for kw in (dict(sliding_window=0), dict(sliding_window=8, sink_tokens=-1)):
        with pytest.raises(ValueError):
            FastestFlashStreamingGQA(256, 4, 2, **kw)
    dec = StreamingDecoder(_module(max_len=64).eval(), max_pages=20, page_size=16)
    x = torch.randn(1, 64, 256, device="cuda", dtype=torch.bfloat16)
    dec.prefill(x, [0])
    with pytest.raises(ValueError):  # a context already
        dec.prefill(x, [0])
    with pytest.raises(ValueError):  # past the rotary tables
        dec.step(x[:, :1], [0])
    with pytest.raises(ValueError):  # a sequence twice in a step
        dec.step(x[:, :1].expand(2, -1, -1), [0, 0])
    full = StreamingDecoder(_module().eval(), max_pages=4, page_size=16)
    full.prefill(x, [0])
    with pytest.raises(RuntimeError):  # no page for the next token: nothing has changed
        full.step(x[:, :1], [0])
    assert dec.cache.position(0) == 64 and full.cache.position(0) == 64
