"""Derivatives through apply_rotary beyond the first, without a GPU: the launch
is replaced by the same rotation on the host, which autograd does not see
either.  The rotation is linear, so second derivatives through it are exact up
to the rounding of fp64 sums."""
import pytest
import torch

from fastest_flash_attention_b200 import rotary


def _turn(x, cos, sin, pos, inverse):
    c, s = cos[pos.long()].double(), sin[pos.long()].double() * (-1 if inverse else 1)
    h = c.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


@pytest.fixture
def host_rotation(monkeypatch):
    def rotate(q, k, cos, sin, pos, layout, inverse):
        with torch.no_grad():
            return tuple(None if t is None else _turn(t.detach(), cos, sin, pos, inverse) for t in (q, k))
    monkeypatch.setattr(rotary, "_rotate", rotate)
    monkeypatch.setattr(rotary._lib, "require_cuda", lambda *ts: None)
    monkeypatch.setitem(rotary._lib.IN_DTYPE_CODE, torch.float64, 0)


def _inputs():
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(2, h, 5, 8, generator=g, dtype=torch.float64, requires_grad=True) for h in (3, 1))
    return q, k, *rotary.rotary_tables(6, 9, device="cpu")


@pytest.mark.parametrize("with_k", [True, False])
def test_second_derivatives(host_rotation, with_k):
    q, k, cos, sin = _inputs()
    ts = (q, k) if with_k else (q,)

    def f(*ts):
        a, b = rotary.apply_rotary(ts[0], ts[1] if with_k else None, cos, sin, 2)
        return (a ** 3).sum() + (0 if b is None else (b ** 3).sum())
    assert torch.autograd.gradcheck(f, ts)
    assert torch.autograd.gradgradcheck(f, ts)


def test_gradient_of_one_output_alone(host_rotation):
    q, k, cos, sin = _inputs()
    a, b = rotary.apply_rotary(q, k, cos, sin, 2)
    dq, dk = torch.autograd.grad((b ** 2).sum(), (q, k), create_graph=True, allow_unused=True)
    assert dq is None or not bool(dq.any())
    torch.testing.assert_close(dk, 2 * k)  # a rotation keeps the norm, 2^-24 in the tables
    torch.testing.assert_close(torch.autograd.grad(dk.sum(), k)[0], torch.full_like(k, 2.0))


def test_forward_mode_is_refused_not_dropped(host_rotation):
    """A dual tensor requires no gradient; its tangent must not vanish."""
    from torch.autograd import forward_ad
    q, k, cos, sin = (t.detach() for t in _inputs())
    with forward_ad.dual_level():
        for a, b in ((forward_ad.make_dual(q, q), None), (forward_ad.make_dual(q, q), k), (q, forward_ad.make_dual(k, k))):
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                rotary.apply_rotary(a, b, cos, sin, 2)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                rotary.apply_rotary(a, b, cos, sin, 2)
        rotary.apply_rotary(q, k, cos, sin, 2)
