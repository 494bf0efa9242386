"""Rotary positions on the sm_100a kernels: tables, the rotation of queries and
keys with its gradient, and its serving form fused with the append to a paged
KV cache.

The reference has rotary positions only inside its MLA module, as a chain of
torch operations (modules/flash_mla.py:29-52, half-split, no scaling); these
functions serve every attention of this package, in both pair layouts, on part
of the head, and for contexts past the trained length.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd import Function, forward_ad

from . import _lib

_LAYOUTS = {"half": 0, "interleaved": 1}
_POS64 = {torch.int32: 0, torch.int64: 1}


def rotary_tables(dim: int, max_len: int, base: float = 10000.0, *, scaling: Optional[str] = None,
                  factor: float = 1.0, original_max_len: Optional[int] = None, beta_fast: float = 32.0,
                  beta_slow: float = 1.0, device: torch.device | str = "cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [max_len, dim / 2], for positions 0 .. max_len - 1.

    Angle i of position p is p * base^(-2 i / dim), computed in 64 bits and
    rounded once, so long positions lose nothing.  ``scaling`` stretches the
    angles by ``factor`` for contexts past the trained length:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised to base * factor^(dim / (dim - 2)), which
      leaves the fastest pair as it is and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times within
      ``original_max_len`` keep their frequency, those that turn less than
      ``beta_slow`` times are divided by ``factor``, a linear ramp between;
      the tables carry the method's attention factor 0.1 ln(factor) + 1.
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary dim must be even and positive, got {dim}")
    if max_len <= 0:
        raise ValueError(f"max_len must be positive, got {max_len}")
    if factor <= 0:
        raise ValueError(f"factor must be positive, got {factor}")
    mscale = 1.0
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs a rotary dim above 2")
        base = base * factor ** (dim / (dim - 2))
    inv = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if not original_max_len:
            raise ValueError("yarn scaling needs original_max_len")

        def pair_of(turns: float) -> float:  # index of the pair that turns so often within original_max_len
            return dim * math.log(original_max_len / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(pair_of(beta_fast)), 0)
        hi = min(math.ceil(pair_of(beta_slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
        mscale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown rotary scaling {scaling!r} (None, 'linear', 'ntk', 'yarn')")
    ang = torch.arange(max_len, dtype=torch.float64)[:, None] * inv[None, :]
    return ((ang.cos() * mscale).to(device, torch.float32), (ang.sin() * mscale).to(device, torch.float32))


def _check_tables(cos: torch.Tensor, sin: torch.Tensor, D: int, layout: str) -> int:
    """The rotated width; raises for tables or a layout the kernels do not take."""
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown rotary layout {layout!r} ('half' or 'interleaved')")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be fp32 [positions, rotary_dim / 2] tables of one shape")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin tables must be contiguous")
    rot = 2 * cos.shape[1]
    if rot == 0 or rot > D or cos.shape[0] == 0:
        raise ValueError(f"rotary dim {rot} does not fit head dim {D} (or the tables are empty)")
    return rot


def _unit_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _rotate(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor,
            layout: int, inverse: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """One launch over q [B, Hq, S, D] and, where given, k [B, Hkv, S, D]."""
    B, Hq, S, D = q.shape
    q = _unit_last(q)
    qo = torch.empty_like(q)
    qs, qd = _lib.three(q), _lib.three(qo)
    if k is not None:
        k = _unit_last(k)
        ko = torch.empty_like(k)
        Hkv, kptr, koptr = k.shape[1], k.data_ptr(), ko.data_ptr()
        ks, kd = _lib.three(k), _lib.three(ko)
    else:
        ko, Hkv, kptr, koptr, ks, kd = None, 0, None, None, None, None
    with _lib.device_of(q):
        st = _lib.direct().ffa_rotary(
            q.data_ptr(), qs, qo.data_ptr(), qd, kptr, ks, koptr, kd, cos.data_ptr(), sin.data_ptr(), cos.shape[0],
            pos.data_ptr(), _POS64[pos.dtype], pos.stride(0) if pos.dim() == 2 else 0, _lib.IN_DTYPE_CODE[q.dtype],
            B, S, Hq, Hkv, D, 2 * cos.shape[1], layout, int(inverse), _lib.err_ptr(q),
            _lib.stream_of(q))
    _lib.check(st, "ffa_rotary")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(q.device)
    return qo, ko


class RotaryFunc(Function):
    """Autograd function of apply_rotary: the gradient of a rotation is the
    rotation by the negative angle (the transpose, with scaled tables too),
    itself through this function where it will be differentiated again."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, pos, layout, inverse):
        ctx.save_for_backward(cos, sin, pos)
        ctx.layout, ctx.inverse = layout, inverse
        ctx.set_materialize_grads(False)
        return _rotate(q, k, cos, sin, pos, layout, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        first, second = (dq, dk) if dq is not None else (dk, None)
        if first is None:
            return (None,) * 7
        a, b = _rotation(first, second, *ctx.saved_tensors, ctx.layout, not ctx.inverse)
        return (a, b) + (None,) * 5 if dq is not None else (None, a) + (None,) * 5


def _rotation(q, k, cos, sin, pos, layout: int, inverse: bool):
    """The rotation, through autograd where an input is part of a graph or may
    carry a tangent (which the function refuses), and only there: it costs host time."""
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
            or forward_ad._current_level >= 0):
        return RotaryFunc.apply(q, k, cos, sin, pos, layout, inverse)
    return _rotate(q, k, cos, sin, pos, layout, inverse)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
                 positions: Union[torch.Tensor, int] = 0, *, layout: str = "half"
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotate q [B, Hq, S, D] and k [B, Hkv, S, D] (or None) by their positions,
    in one launch; differentiable in q and k.

    cos, sin: fp32 tables [positions, rotary_dim / 2] (``rotary_tables``); the
    first rotary_dim values of each head turn, the rest pass through.
    positions: int32 / int64 [S] or [B, S] on the device, or the position of
    the first token.  layout: pairs (i, i + rotary_dim / 2) for "half",
    (2 i, 2 i + 1) for "interleaved".  fp16, bf16 or fp32; any strides.  A
    position outside the tables leaves its token unturned and sets the device
    error word.
    """
    _lib.require_cuda(q, k, cos, sin)
    if q.dim() != 4:
        raise ValueError(f"q must be [B, H, S, D], got {tuple(q.shape)}")
    B, _, S, D = q.shape
    if k is not None and (k.dim() != 4 or k.shape[0] != B or k.shape[2] != S or k.shape[3] != D
                          or k.dtype != q.dtype):
        raise ValueError(f"incompatible q/k {tuple(q.shape)} {q.dtype} and {tuple(k.shape)} {k.dtype}")
    if q.dtype not in _lib.IN_DTYPE_CODE:
        raise ValueError(f"apply_rotary takes fp16, bf16 or fp32, got {q.dtype}")
    _check_tables(cos, sin, D, layout)
    if isinstance(positions, int):
        if positions < 0 or positions + S > cos.shape[0]:
            raise ValueError(f"positions [{positions}, {positions + S}) are outside the tables' {cos.shape[0]}")
        positions = torch.arange(positions, positions + S, dtype=torch.int32, device=q.device)
    _lib.require_cuda(q, positions)
    if positions.dtype not in _POS64 or tuple(positions.shape) not in ((S,), (B, S)):
        raise ValueError(f"positions must be int32 or int64 [S] or [B, S], got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    return _rotation(q, k, cos, sin, _unit_last(positions), _LAYOUTS[layout], False)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                  layout: str = "half") -> torch.Tensor:
    """Serving form, one launch for T new tokens: returns q rotated, and writes
    the rotated k and v into their slots of the page pools.

    q [T, Hq, D]; k, v [T, Hkv, D] (any strides, e.g. slices of one stacked
    projection); positions int32 / int64 [T]; slots int32 [T] = page *
    page_size + offset, distinct (one outside the pool writes nothing: padding
    tokens); k_pages, v_pages [P, Hkv, page_size, D] contiguous.
    """
    _lib.require_cuda(q, k, v, cos, sin, positions, slots, k_pages, v_pages)
    if q.dim() != 3 or k.dim() != 3 or k_pages.dim() != 4:
        raise ValueError("rotary_append takes q [T, Hq, D], k / v [T, Hkv, D] and pools [P, Hkv, page_size, D]")
    T, Hq, D = q.shape
    P, Hkv, page_size, Dp = k_pages.shape
    if k.shape != v.shape or tuple(k.shape) != (T, Hkv, D) or Dp != D or v_pages.shape != k_pages.shape:
        raise ValueError(f"incompatible shapes q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)} pools "
                         f"{tuple(k_pages.shape)} {tuple(v_pages.shape)}")
    dt = q.dtype
    if dt not in _lib.IN_DTYPE_CODE or not (k.dtype == v.dtype == k_pages.dtype == v_pages.dtype == dt):
        raise ValueError("rotary_append needs q, k, v and both pools of one dtype (fp16, bf16 or fp32)")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("page pools must be contiguous")
    rot = _check_tables(cos, sin, D, layout)
    if positions.dtype not in _POS64 or positions.dim() != 1 or positions.shape[0] != T:
        raise ValueError(f"positions must be int32 or int64 [T], got {positions.dtype} {tuple(positions.shape)}")
    if slots.dtype != torch.int32 or slots.dim() != 1 or slots.shape[0] != T:
        raise ValueError(f"slots must be int32 [T], got {slots.dtype} {tuple(slots.shape)}")
    q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
    positions, slots = _unit_last(positions), _unit_last(slots)
    out = q.new_empty((T, Hq, D))
    with _lib.device_of(q):
        st = _lib.direct().ffa_rotary_append(
            q.data_ptr(), q.stride(), out.data_ptr(), (Hq * D, D), k.data_ptr(), k.stride(), v.data_ptr(), v.stride(),
            cos.data_ptr(),
            sin.data_ptr(), cos.shape[0], positions.data_ptr(), _POS64[positions.dtype], slots.data_ptr(),
            k_pages.data_ptr(), v_pages.data_ptr(), _lib.IN_DTYPE_CODE[dt], T, Hq, Hkv, D, rot, _LAYOUTS[layout],
            page_size, P, _lib.err_ptr(q), _lib.stream_of(q))
    _lib.check(st, "ffa_rotary_append")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(q.device)
    return out
