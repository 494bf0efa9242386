"""Attention with sinks on the storage orders that modules and caches hand it:
bit for bit what the [B, S, H, D] storage of the other tests gives (strides
change addresses, not the order of any sum)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _run(q, k, v, do, **kw):
    from fastest_flash_attention_b200 import fastest_flash_attn_forward, fastest_flash_attn_func
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = fastest_flash_attn_func(q, k, v, **kw)
    _, lse = fastest_flash_attn_forward(q.detach(), k.detach(), v.detach(), return_lse=True, **kw)
    return (o, lse) + torch.autograd.grad(o, (q, k, v), do)


def _stored(ts, storage):
    """The same values as [B, H, S, D] views of another storage."""
    B, S = ts[0].shape[0], ts[0].shape[2]
    if storage == "bhsd":
        return [t.contiguous() for t in ts]
    if storage == "padded":  # longer rows, more heads and tokens around them
        out = []
        for t in ts:
            base = torch.full((B, S + 3, t.shape[1] + 1, t.shape[3] + 8), float("nan"), dtype=t.dtype, device="cuda")
            view = base[:, 1:1 + S, :t.shape[1], :t.shape[3]].transpose(1, 2)
            out.append(view.copy_(t))
        return out
    widths = [t.shape[1] * t.shape[3] for t in ts]  # slices of one stacked projection
    y = torch.empty(B, S, sum(widths), dtype=ts[0].dtype, device="cuda")
    return [s.view(B, S, t.shape[1], t.shape[3]).transpose(1, 2).copy_(t) for s, t in zip(y.split(widths, -1), ts)]


@pytest.mark.parametrize("storage", ["bhsd", "padded", "stacked"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,Dv,window,sinks", [
    (2, 4, 2, 300, 128, 128, 64, 4), (1, 4, 1, 777, 64, 64, 100, 130), (2, 2, 2, 200, 40, 24, 30, 3),
    (1, 4, 2, 400, 192, 128, 90, 5), (1, 2, 1, 333, 136, 72, 128, 4), (3, 1, 1, 1, 64, 64, 1, 1)])
def test_storage_orders(B, Hq, Hkv, S, D, Dv, window, sinks, dtype, storage):
    g = torch.Generator(device="cuda").manual_seed(S + D)
    ts = [torch.randn(B, S, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
          for h, d in ((Hq, D), (Hkv, D), (Hkv, Dv), (Hq, Dv))]
    kw = dict(causal=True, sliding_window=window, sink_tokens=sinks)
    want = _run(*ts, **kw)
    other = _stored(ts, storage)
    assert all(torch.equal(a, b) for a, b in zip(other, ts))
    for a, b in zip(_run(*other, **kw), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cached,new", [(1, 1), (250, 1), (250, 77), (100, 300)])
def test_cached_keys_before_the_new_ones(cached, new, dtype):
    """kv_cache= puts the cached keys first; the queries are the last positions."""
    from fastest_flash_attention_b200 import fastest_flash_attn_forward
    from fastest_flash_attention_b200.attention import flash_fwd
    g = torch.Generator(device="cuda").manual_seed(cached)
    k, v = (torch.randn(2, 2, cached + new, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(2, 4, new, 64, generator=g, device="cuda").to(dtype)
    o, lse = fastest_flash_attn_forward(q, k[:, :, cached:], v[:, :, cached:], causal=True, sliding_window=60, sink_tokens=5,
                                        kv_cache=(k[:, :, :cached], v[:, :, :cached]), return_lse=True)
    want, want_lse = flash_fwd(q, k, v, scale=0.125, causal=True, q_offset=cached, window=60, sink=5)
    assert torch.equal(o, want) and torch.equal(lse[..., 0], want_lse)
    i = torch.arange(new, device="cuda")[:, None] + cached
    j = torch.arange(cached + new, device="cuda")[None]
    seen = (j <= i) & ((j > i - 60) | (j < 5))
    kk, vv = (t.double().repeat_interleave(2, 1) for t in (k, v))
    exact = torch.softmax((q.double() @ kk.transpose(-1, -2) * 0.125).masked_fill(~seen, -float("inf")), -1) @ vv
    # P and O rounded once each (2^-8 in bf16), or fp32 sums of 65 terms
    tol = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5
    assert float((o.double() - exact).norm()) <= tol * float(exact.norm())
