"""Several new tokens of each request against its cached pages, on the sm_100a
tensor cores.

The reference runs them by gathering each sequence's pages into a contiguous
tensor (ops/kv_cache.py:208-232) and calling the forward with a cache
(ops/attention_forward.py:80-89).  ``paged_prefill`` attends straight from the
page pool, all requests of a batch in one launch: chunks of prompts, drafted
tokens to verify and single tokens side by side.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch
from torch.autograd import Function, forward_ad

from . import _lib


def check_pools(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, what: str) -> tuple:
    """(tokens, Hq, D, P, Hkv, page_size) of q [tokens, Hq, D] and the pools [P, Hkv, page_size, D]; raises unless
    they fit the tensor-core kernels over pages."""
    qs, ks = q.shape, k_pages.shape
    if len(qs) != 3 or len(ks) != 4:
        raise ValueError(f"q must be [tokens, Hq, D] and the pools [P, Hkv, page_size, D], got {tuple(qs)} and "
                         f"{tuple(ks)}")
    T, Hq, D = qs
    P, Hkv, page_size, Dk = ks
    if Dk != D or v_pages.shape != ks:
        raise ValueError("q / page pool head dims disagree")
    if P == 0 or Hkv == 0 or Hq == 0 or Hq % Hkv or Hq // Hkv > 128:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key/value heads ({Hkv}), at most 128 times")
    if D == 0 or D % 8 or D > 128:
        raise ValueError(f"{what} takes head dims up to 128 that are multiples of 8, got {D}")
    if page_size == 0 or page_size % 8:
        raise ValueError(f"{what} takes page sizes that are multiples of 8, got {page_size}")
    dt = q.dtype
    if dt not in _lib.DTYPE_CODE or k_pages.dtype is not dt or v_pages.dtype is not dt:
        raise ValueError(f"{what} needs fp16/bf16 q and pages of the same dtype")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("page pools must be contiguous")
    return T, Hq, D, P, Hkv, page_size


def check_scale(scale: Optional[float], softcap: Optional[float], D: int) -> tuple:
    """(scale, softcap) as the kernels take them; both positive (a row's maximum is found before either is applied)."""
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not 0.0 < scale < math.inf or not 0.0 <= softcap < math.inf:
        raise ValueError(f"scale and softcap must be positive, got {scale} and {softcap}")
    return scale, softcap


def tma_rows(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, D] as TMA reads it: contiguous heads, other strides and the base multiples of 16 bytes."""
    sr, sh, sd = t.stride()
    if sd != 1 or (sr | sh) % 8 or sr <= 0 or sh <= 0 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def heads_apart(t: torch.Tensor) -> bool:
    """Whether no two heads of t [tokens, heads, D], D contiguous, share memory."""
    (T, H, D), (st, sh) = t.shape, t.stride()[:2]
    if (T > 1 and st < D) or (H > 1 and sh < D):
        return False
    if T < 2 or H < 2 or st >= (H - 1) * sh + D or sh >= (T - 1) * st + D:
        return True
    # neither axis lies within the other: head h of a token against head 0 of those whose heads begin next to it
    return all(n >= T or abs(h * sh - n * st) >= D for h in range(1, H) for n in (h * sh // st, h * sh // st + 1))


class _NoGradient(Function):
    """The results of a call that has no backward pass; a gradient that reaches them is refused, not left out."""

    @staticmethod
    def forward(ctx, what, results, *inputs):
        ctx.what = what
        return results  # (no inputs of this function, so not views of them)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} has no backward pass")


def without_gradient(what: str, o: torch.Tensor, lse: Optional[torch.Tensor], q: torch.Tensor, k_pages: torch.Tensor,
                     v_pages: torch.Tensor, given: bool = False) -> tuple:
    """(o, lse), which refuse a gradient (or a tangent) where an input is part of a graph.  given: o is the caller's
    own tensor, which does not become part of one."""
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled() \
            or forward_ad._current_level >= 0:
        return _NoGradient.apply(what, (o.detach() if given else o, lse), q, k_pages, v_pages)
    return o, lse


@functools.lru_cache(maxsize=1024)
def _workspace(*sizes: int) -> int:
    return _lib.load().ffa_paged_prefill_workspace_size(*sizes)


def paged_prefill(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                  ctx_lens: torch.Tensor, query_starts: torch.Tensor, *, scale: Optional[float] = None,
                  softcap: Optional[float] = None, return_lse: bool = False, max_ctx: Optional[int] = None,
                  out: Optional[torch.Tensor] = None):
    """Causal attention of each request's last tokens over its pages.

    q [T, Hq, D]: request r's queries are rows [query_starts[r],
    query_starts[r + 1]), the last of its ctx_lens[r] tokens, whose keys and
    values are in the pages already; query i of n sees the first
    ctx_lens[r] - n + i + 1 tokens.  k_pages / v_pages [P, Hkv, page_size, D]
    contiguous, page_size a multiple of 8; block_table [R, max_pages],
    ctx_lens [R], query_starts [R + 1] int32 / int64 (``assign_slots`` gives all
    three).  max_ctx: the longest context, if known (it only chooses how
    contexts are split, and with that the last bits; without it they are split
    as if they filled the table).  A value that is NaN or infinite reaches the
    queries that share a tile with one that sees it, as in the dense forward; a
    key only those that see it.  Returns o [T, Hq, D] and, if requested, lse [T, Hq]
    fp32 (natural log); ``out`` takes o in a given tensor.  Rows that belong to
    no request are not written.  There is no backward pass: a gradient that
    reaches the results raises.

    query_starts that decrease or pass T, a request with more queries than
    tokens, a length past the table and a page id outside the pool set the
    device error word.
    """
    _lib.require_cuda(q, k_pages, v_pages, block_table, ctx_lens, query_starts, out)
    T, Hq, D, P, Hkv, page_size = check_pools(q, k_pages, v_pages, "paged_prefill")
    table = block_table.shape
    if len(table) != 2 or table[1] == 0 or ctx_lens.shape != (table[0],) or query_starts.shape != (table[0] + 1,):
        raise ValueError(f"block_table must be [R, max_pages], ctx_lens [R] and query_starts [R + 1], got "
                         f"{tuple(table)}, {tuple(ctx_lens.shape)} and {tuple(query_starts.shape)}")
    if max_ctx is not None and max_ctx < 0:
        raise ValueError(f"max_ctx must not be negative, got {max_ctx}")
    scale, softcap = check_scale(scale, softcap, D)
    R, width = table
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or (out.stride(0) | out.stride(1)) % 8 \
            or out.data_ptr() % 16 or not heads_apart(out):
        raise ValueError("out must be like q, with heads apart and contiguous, other strides and the base multiples of "
                         "16 bytes")
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    if T == 0 or R == 0:
        return (out, lse) if return_lse else out
    bt, lens, starts = _lib.int32(block_table), _lib.int32(ctx_lens), _lib.int32(query_starts)
    q = tma_rows(q)
    most = min(width * page_size, 2 ** 31 - 1)
    ctx = most if max_ctx is None else min(max_ctx, most)
    ws_bytes = _workspace(R, T, Hq, Hkv, D, ctx)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    with _lib.device_of(q):
        st = _lib.direct().ffa_paged_prefill(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), bt.data_ptr(), lens.data_ptr(), starts.data_ptr(),
            out.data_ptr(), lse.data_ptr() if return_lse else None, _lib.DTYPE_CODE[q.dtype], R, T, Hq, Hkv, D, P,
            page_size, width, q.stride()[:2], out.stride()[:2], scale, softcap, ctx,
            ws.data_ptr() if ws_bytes else None, ws_bytes, _lib.err_ptr(q), _lib.stream_of(q))
    _lib.check(st, "ffa_paged_prefill")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(q.device)
    out, lse = without_gradient("paged_prefill", out, lse, q, k_pages, v_pages, given=given)
    return (out, lse) if return_lse else out
