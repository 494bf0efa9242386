"""Refusals of prefix_decode that need no GPU."""
import math

import pytest
import torch

import fastest_flash_attention_b200 as ffa


def test_entry_point_refuses_sizes_that_mean_nothing():
    from fastest_flash_attention_b200 import _lib
    lib, p, s = _lib.load(), 4096, _lib.i64arr(512, 64)  # nothing is dereferenced: the sizes are refused first
    good = dict(dtype=1, R=2, G=1, Hq=8, Hkv=2, D=64, P=4, page=16, width=2, qs=s, os=s, scale=1.0, mp=32, mo=0, q=p,
                kp=p, vp=p, bt=p, ln=p, st=p, pf=p, out=p, ws=p, bytes=1 << 30)

    def call(**kw):
        a = dict(good, **kw)
        return lib.ffa_prefix_decode(a["q"], a["kp"], a["vp"], a["bt"], a["ln"], a["st"], a["pf"], a["out"], None,
                                     a["dtype"], a["R"], a["G"], a["Hq"], a["Hkv"], a["D"], a["P"], a["page"],
                                     a["width"], a["qs"], a["os"], a["scale"], 0.0, a["mp"], a["mo"], a["ws"],
                                     a["bytes"], None, None)
    bad = (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
    for kw in (dict(R=-1), dict(G=-1), dict(Hq=7), dict(Hkv=0), dict(Hq=258), dict(D=0), dict(D=60), dict(D=136),
               dict(P=0), dict(page=0), dict(page=12), dict(width=0), dict(P=2 ** 30), dict(width=2 ** 30),
               dict(scale=0.0), dict(scale=math.nan), dict(dtype=2), dict(mp=-1), dict(mo=-1), dict(q=None),
               dict(kp=None), dict(vp=None), dict(bt=None), dict(ln=None), dict(st=None), dict(pf=None), dict(out=None),
               dict(q=p + 2), dict(vp=p + 2), dict(qs=_lib.i64arr(512, 60)), dict(qs=None), dict(os=None)):
        assert call(**kw) in bad, kw
    assert call(R=0) == _lib.FFA_OK
    # a prefix long enough to be read once for the group needs its workspace; a short one needs none
    for kw in (dict(ws=None), dict(bytes=100), dict(ws=p + 8)):
        assert call(mp=50000, **kw) == _lib.FFA_ERR_WORKSPACE
    assert lib.ffa_prefix_decode_workspace_size(2, 1, 8, 2, 64, 50000) > 0
    assert lib.ffa_prefix_decode_workspace_size(2, 1, 8, 2, 64, 32) == 0
    for sizes in ((0, 1, 8, 2, 64, 9), (2, 0, 8, 2, 64, 9), (2, 1, 7, 2, 64, 9), (2, 1, 8, 0, 64, 9),
                  (2, 1, 8, 2, 0, 9), (2, 1, 8, 2, 64, -1), (2, 1, 258, 2, 64, 9)):
        assert lib.ffa_prefix_decode_workspace_size(*sizes) == 0


def test_arguments_are_refused(monkeypatch):
    from fastest_flash_attention_b200 import _lib
    q, pool = torch.zeros(4, 8, 64).half(), torch.zeros(3, 2, 16, 64).half()
    bt, ln, st, pf = torch.zeros(4, 3).int(), torch.zeros(4).int(), torch.zeros(2).int(), torch.zeros(1).int()
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.prefix_decode(q, pool, pool, bt, ln, st, pf)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", lambda: pytest.fail("the call was not refused"))
    good = dict(q=q, kp=pool, vp=pool, bt=bt, ln=ln, st=st, pf=pf)
    for kw in (dict(q=q[0]), dict(q=q[:, :7]), dict(q=q.float()), dict(q=q[..., :60]), dict(kp=pool[0]),
               dict(vp=pool[:, :1]), dict(kp=pool.bfloat16()), dict(kp=pool.transpose(1, 2), vp=pool.transpose(1, 2)),
               dict(kp=pool[:, :, :12].contiguous(), vp=pool[:, :, :12].contiguous()), dict(bt=bt[:3]),
               dict(bt=bt[:, :0]), dict(bt=bt[0]), dict(ln=ln[:3]), dict(st=st[:1]), dict(st=st[:, None]),
               dict(pf=pf[:0]), dict(pf=pf[0])):
        a = dict(good, **kw)
        with pytest.raises(ValueError):
            ffa.prefix_decode(a["q"], a["kp"], a["vp"], a["bt"], a["ln"], a["st"], a["pf"])
    for kw in (dict(scale=0.0), dict(scale=math.nan), dict(softcap=-1.0), dict(max_prefix=-1), dict(max_own=-1)):
        with pytest.raises(ValueError):
            ffa.prefix_decode(q, pool, pool, bt, ln, st, pf, **kw)
