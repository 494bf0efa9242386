"""Decoding of requests that share a prefix (a system prompt, the samples of one
prompt, questions on one document), the prefix computed once for all of them (no
counterpart in the reference).

``paged_decode`` reads a shared page once for every request.  ``prefix_decode``
reads it once for the group: one launch attends the prefix with the query heads
of all its requests as the rows of tensor-core products, a second, overlapping
one attends each request's own tokens and joins the two by their LSE (or leaves
that to a third, where the prefix leaves SMs idle for long).  Where there is little
to share, one launch attends each request's tokens instead.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from .prefill import check_pools, check_scale, tma_rows, without_gradient


@functools.lru_cache(maxsize=1024)
def _workspace(*sizes: int) -> int:
    return _lib.load().ffa_prefix_decode_workspace_size(*sizes)


def prefix_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                  ctx_lens: torch.Tensor, group_starts: torch.Tensor, prefix_lens: torch.Tensor, *,
                  scale: Optional[float] = None, softcap: Optional[float] = None, return_lse: bool = False,
                  max_prefix: Optional[int] = None, max_own: Optional[int] = None):
    """Decode attention for R requests, groups of which share their first tokens.

    q [R, Hq, D]; k_pages / v_pages [P, Hkv, page_size, D] contiguous, page_size
    a multiple of 8; block_table [R, max_pages], ctx_lens [R] as
    ``paged_decode``.  Requests [group_starts[g], group_starts[g + 1]) hold the
    same first prefix_lens[g] tokens, which are read through the table row of
    the group's first request that is long enough; the rest of each request
    through its own row.  group_starts [G + 1] and prefix_lens [G] int32 /
    int64 on the device; a request shorter than its group's prefix, or in no
    group, is computed by itself.  max_prefix, max_own: the longest prefix and
    the most tokens of a request behind it, if known.  They only choose how the
    work is split, and with that the last bits; but without them a prefix is
    split as if it filled the table, which takes 1.5 to 4 times as long where
    the table is four to sixteen times as wide.  Returns o [R, Hq, D] (q's
    dtype) and, if requested, lse [R, Hq] fp32 (natural log; a request without
    tokens gets 0 and -inf).  There is no backward pass: a gradient that reaches
    the results raises.

    Boundaries that decrease or pass R, a length past the table and a page id
    outside the pool set the device error word.
    """
    _lib.require_cuda(q, k_pages, v_pages, block_table, ctx_lens, group_starts, prefix_lens)
    R, Hq, D, P, Hkv, page_size = check_pools(q, k_pages, v_pages, "prefix_decode")
    table, groups = block_table.shape, prefix_lens.shape
    if len(table) != 2 or table[0] != R or table[1] == 0 or ctx_lens.shape != (R,):
        raise ValueError(f"block_table must be [{R}, max_pages] and ctx_lens [{R}], got {tuple(table)} and "
                         f"{tuple(ctx_lens.shape)}")
    if len(groups) != 1 or group_starts.shape != (groups[0] + 1,):
        raise ValueError(f"group_starts must be [G + 1] and prefix_lens [G], got {tuple(group_starts.shape)} and "
                         f"{tuple(groups)}")
    if (max_prefix or 0) < 0 or (max_own or 0) < 0:
        raise ValueError(f"max_prefix and max_own must not be negative, got {max_prefix} and {max_own}")
    scale, softcap = check_scale(scale, softcap, D)
    width, groups = table[1], groups[0]
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((R, Hq), dtype=torch.float32) if return_lse else None
    if R == 0:
        return (out, lse) if return_lse else out
    bt, lens = _lib.int32(block_table), _lib.int32(ctx_lens)
    starts, prefixes = _lib.int32(group_starts), _lib.int32(prefix_lens)
    q = tma_rows(q)
    most = min(width * page_size, 2 ** 31 - 1)
    prefix = most if max_prefix is None else min(max_prefix, most)
    ws_bytes = _workspace(R, groups, Hq, Hkv, D, prefix)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    with _lib.device_of(q):
        st = _lib.direct().ffa_prefix_decode(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), bt.data_ptr(), lens.data_ptr(), starts.data_ptr(),
            prefixes.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, _lib.DTYPE_CODE[q.dtype], R,
            groups, Hq, Hkv, D, P, page_size, width, q.stride()[:2], (Hq * D, D), scale, softcap, prefix,
            min(max_own or 0, most), ws.data_ptr() if ws_bytes else None, ws_bytes, _lib.err_ptr(q), _lib.stream_of(q))
    _lib.check(st, "ffa_prefix_decode")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(q.device)
    out, lse = without_gradient("prefix_decode", out, lse, q, k_pages, v_pages)
    return (out, lse) if return_lse else out
