"""Refusals of paged_prefill that need no GPU."""
import math

import pytest
import torch

import fastest_flash_attention_b200 as ffa


def test_entry_point_refuses_sizes_that_mean_nothing():
    from fastest_flash_attention_b200 import _lib
    lib, p, s = _lib.load(), 4096, _lib.i64arr(512, 64)  # nothing is dereferenced: the sizes are refused first
    good = dict(dtype=1, R=1, T=2, Hq=8, Hkv=2, D=64, P=4, page=16, width=2, qs=s, os=s, scale=1.0, cap=0.0, ctx=32,
                q=p, kp=p, vp=p, bt=p, ln=p, st=p, out=p)

    def call(**kw):
        a = dict(good, **kw)
        return lib.ffa_paged_prefill(a["q"], a["kp"], a["vp"], a["bt"], a["ln"], a["st"], a["out"], None, a["dtype"],
                                     a["R"], a["T"], a["Hq"], a["Hkv"], a["D"], a["P"], a["page"], a["width"], a["qs"],
                                     a["os"], a["scale"], a["cap"], a["ctx"], None, 0, None, None)
    bad = (_lib.FFA_ERR_INVALID_ARG, _lib.FFA_ERR_UNSUPPORTED)
    for kw in (dict(R=-1), dict(T=-1), dict(Hq=7), dict(Hkv=0), dict(Hq=0), dict(Hq=258, Hkv=2), dict(D=0), dict(D=60),
               dict(D=136), dict(P=0), dict(page=0), dict(page=12), dict(width=0), dict(P=2 ** 30), dict(width=2 ** 30),
               dict(T=2 ** 30), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(dtype=2), dict(ctx=-1),
               dict(q=None), dict(kp=None), dict(vp=None), dict(bt=None), dict(ln=None), dict(st=None), dict(out=None),
               dict(q=p + 2), dict(kp=p + 2), dict(out=p + 8), dict(qs=_lib.i64arr(512, 60)), dict(qs=None),
               dict(os=None), dict(os=_lib.i64arr(4, 64)), dict(qs=_lib.i64arr(-512, 64))):
        assert call(**kw) in bad, kw
    assert call(R=0) == call(T=0) == _lib.FFA_OK
    # a split context needs its workspace
    assert call(ctx=5000, width=400) == _lib.FFA_ERR_WORKSPACE
    assert lib.ffa_paged_prefill_workspace_size(1, 2, 8, 2, 64, 5000) > 0
    for sizes in ((0, 2, 8, 2, 64, 9), (1, 0, 8, 2, 64, 9), (1, 2, 0, 2, 64, 9), (1, 2, 8, 0, 64, 9),
                  (1, 2, 7, 2, 64, 9), (1, 2, 8, 2, 0, 9), (1, 2, 8, 2, 64, -1), (1, 2, 258, 2, 64, 9),
                  (1, 2, 8, 2, 64, 0), (1, 2, 8, 2, 64, 128)):
        assert lib.ffa_paged_prefill_workspace_size(*sizes) == 0
    assert lib.ffa_paged_prefill_workspace_size(1, 1, 8, 2, 64, 2 ** 31 - 1) < 2 ** 20


def test_arguments_are_refused(monkeypatch):
    from fastest_flash_attention_b200 import _lib
    q, pool = torch.zeros(4, 8, 64).half(), torch.zeros(3, 2, 16, 64).half()
    bt, ln, st = torch.zeros(2, 3).int(), torch.zeros(2).int(), torch.zeros(3).int()
    with pytest.raises(RuntimeError, match="CUDA"):
        ffa.paged_prefill(q, pool, pool, bt, ln, st)
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", lambda: pytest.fail("the call was not refused"))
    good = dict(q=q, kp=pool, vp=pool, bt=bt, ln=ln, st=st)
    for kw in (dict(q=q[0]), dict(q=q[:, :7]), dict(q=q.float()), dict(q=q[..., :60]), dict(kp=pool[0]),
               dict(vp=pool[:, :1]), dict(kp=pool.bfloat16()), dict(vp=pool.bfloat16()),
               dict(kp=pool.transpose(1, 2), vp=pool.transpose(1, 2)), dict(kp=pool[:0], vp=pool[:0]),
               dict(kp=pool[:, :, :12].contiguous(), vp=pool[:, :, :12].contiguous()),
               dict(q=q[..., :60], kp=pool[..., :60].contiguous(), vp=pool[..., :60].contiguous()),
               dict(bt=bt[0]), dict(bt=bt[:, :0]), dict(ln=ln[:1]), dict(st=st[:2])):
        a = dict(good, **kw)
        with pytest.raises(ValueError):
            ffa.paged_prefill(a["q"], a["kp"], a["vp"], a["bt"], a["ln"], a["st"])
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(softcap=-1.0),
               dict(softcap=math.nan), dict(max_ctx=-1), dict(out=torch.zeros(4, 8, 32).half()),
               dict(out=torch.zeros(4, 8, 64)), dict(out=torch.zeros(4, 8, 68).half()[..., :64]),
               dict(out=torch.zeros(4, 64, 8).half().transpose(1, 2))):
        with pytest.raises(ValueError):
            ffa.paged_prefill(q, pool, pool, bt, ln, st, **kw)


def test_an_output_that_overlaps_itself_is_refused(monkeypatch):
    from fastest_flash_attention_b200 import _lib
    q, pool = torch.zeros(4, 8, 64).half(), torch.zeros(3, 2, 16, 64).half()
    bt, ln, st = torch.zeros(2, 3).int(), torch.zeros(2).int(), torch.zeros(3).int()
    monkeypatch.setattr(_lib, "require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "direct", lambda: pytest.fail("the call was not refused"))
    for out in (torch.zeros(1, 8, 64).half().expand(4, 8, 64), torch.zeros(4, 1, 64).half().expand(4, 8, 64),
                torch.zeros(4096).half().as_strided((4, 8, 64), (512, 32, 1))):
        with pytest.raises(ValueError):
            ffa.paged_prefill(q, pool, pool, bt, ln, st, out=out)
