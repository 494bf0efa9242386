"""Second derivatives through attention with sinks, which the kernels do not
have, are refused rather than left out (no GPU: the launches are replaced)."""
import pytest
import torch

from fastest_flash_attention_b200 import attention


def test_second_derivative_is_refused(monkeypatch):
    monkeypatch.setattr(attention, "flash_fwd", lambda q, k, v, **kw: (q.detach() * 2, q.detach()[..., 0]))
    monkeypatch.setattr(attention, "flash_bwd", lambda g, q, k, v, o, lse, **kw: (g * 2, k.detach() * 0, v.detach() * 0))
    q, k, v = (torch.randn(1, 2, 4, 8, requires_grad=True) for _ in range(3))
    out = attention.fastest_flash_attn_func(q, k, v, causal=True, sliding_window=2, sink_tokens=1)
    first, = torch.autograd.grad(out.sum(), q, create_graph=True)
    assert torch.equal(first, torch.full_like(q, 2.0))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad((first ** 2).sum() + (q ** 3).sum(), q)
    out = attention.fastest_flash_attn_func(q, k, v, causal=True, sliding_window=2, sink_tokens=1)
    assert torch.equal(torch.autograd.grad(out.sum(), q)[0], torch.full_like(q, 2.0))
