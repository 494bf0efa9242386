"""Calls over pages have no backward pass: they say so where a gradient would be left out, and run as ever otherwise."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import fastest_flash_attention_b200 as ffa


def _calls(device):
    q, kp, vp = (torch.randn(s, device=device).half() for s in ((3, 4, 64), (6, 2, 16, 64), (6, 2, 16, 64)))

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=device)
    bt, lens = ints([[0, 1], [2, 3], [4, 5]]), ints([20, 17, 31])

    def prefill(q, kp, vp, **kw):
        return ffa.paged_prefill(q, kp, vp, bt, lens, ints([0, 1, 2, 3]), **kw)

    def prefix(q, kp, vp, **kw):
        return ffa.prefix_decode(q, kp, vp, bt, lens, ints([0, 3]), ints([0]), **kw)
    return (q, kp, vp), {"paged_prefill": prefill, "prefix_decode": prefix}


def _stub(monkeypatch):
    from fastest_flash_attention_b200 import _lib

    class Launches:
        def ffa_paged_prefill(self, *a):
            return 0
        ffa_prefix_decode = ffa_paged_prefill
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", Launches)
    monkeypatch.setattr(_lib, "err_ptr", lambda t: 0)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "device_of", lambda t: _lib._HERE)
    monkeypatch.setattr(_lib, "sync_check_enabled", lambda: False)


def _refuses(device):
    inputs, calls = _calls(device)
    for name, call in calls.items():
        for i in range(3):
            args = [x.clone().requires_grad_(i == j) for j, x in enumerate(inputs)]
            o, lse = call(*args, return_lse=True)
            assert o.shape == (3, 4, 64) and lse.shape == (3, 4)
            for loss in (o.float().sum(), lse.sum(), call(*args).float().sum() + sum(x.float().sum() for x in args)):
                with pytest.raises(RuntimeError, match=f"{name} has no backward"):
                    loss.backward()
            o.add_(1)
            with torch.no_grad():  # as ever where none is asked for
                assert not call(*args).requires_grad
            assert not call(*(x.detach() for x in args)).requires_grad
        with fwd.dual_level(), pytest.raises(NotImplementedError):
            call(fwd.make_dual(inputs[0], inputs[0]), *inputs[1:])
        with fwd.dual_level():
            call(*inputs)
    out = torch.empty_like(inputs[0])
    args = [x.clone().requires_grad_() for x in inputs]
    o = calls["paged_prefill"](*args, out=out)
    assert not out.requires_grad and o.data_ptr() == out.data_ptr()
    with pytest.raises(RuntimeError, match="no backward"):
        o.float().sum().backward()
    with torch.no_grad():
        assert calls["paged_prefill"](*args, out=out) is out


def test_gradients_are_refused(monkeypatch):
    _stub(monkeypatch)
    _refuses("cpu")


@pytest.mark.gpu
def test_gradients_are_refused_on_the_device():
    _refuses("cuda")
    inputs, calls = _calls("cuda")
    for call in calls.values():  # the same values either way
        assert torch.equal(call(*(x.clone().requires_grad_() for x in inputs)), call(*inputs))
