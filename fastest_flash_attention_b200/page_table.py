"""Block tables and slot maps built on the GPU from request lengths (no
counterpart in the reference, whose paged cache keeps its tables in Python
lists, ops/kv_cache.py:110-240).

``assign_slots`` takes pages for the new tokens of a batch from a ring of free
ones and gives every token its slot and position; ``release_pages`` puts the
pages of finished requests back.  Both follow the allocation order of
``PagedKVCache`` (first in, first out; requests in batch order), read and write
device tensors alone and synchronise nothing, so a serving step (assign_slots,
rotary_append, paged_prefill or prefix_decode, release_pages) can be captured
in a CUDA graph.  ``DevicePageTable`` keeps the tensors of one pool together.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib


class SlotPlan(NamedTuple):
    """What ``assign_slots`` returns, int32 on the device."""
    slots: torch.Tensor       # [max_tokens] page * page_size + offset; -1 behind the batch's last token
    positions: torch.Tensor   # [max_tokens] position in its request; 0 behind the last token
    starts: torch.Tensor      # [R + 1] request r's new tokens are [starts[r], starts[r + 1])
    ctx_lens: torch.Tensor    # [R] lengths with the new tokens
    free_state: torch.Tensor  # [2] (head, count) of the free pages left


def _check(block_table: torch.Tensor, ctx_lens: torch.Tensor, free_pages: torch.Tensor, free_state: torch.Tensor,
           rows: torch.Tensor, what: str, page_size: int) -> Tuple[int, int, int]:
    table, ring = block_table.shape, free_pages.shape
    if len(table) != 2 or table[1] == 0 or len(ring) != 1 or ring[0] == 0:
        raise ValueError("block_table must be [R, max_pages] and free_pages [num_pages]")
    R, width = table
    if ctx_lens.shape != (R,) or rows.shape != (R,) or free_state.shape != (2,):
        raise ValueError(f"ctx_lens and {what} must be [{R}] and free_state [2], got {tuple(ctx_lens.shape)}, "
                         f"{tuple(rows.shape)} and {tuple(free_state.shape)}")
    for t in (block_table, ctx_lens, free_pages, free_state):
        if t.dtype is not torch.int32 or not t.is_contiguous():
            raise ValueError("block_table, ctx_lens, free_pages and free_state must be contiguous int32 tensors")
    if page_size <= 0:
        raise ValueError(f"page_size must be positive, got {page_size}")
    return R, width, ring[0]


def assign_slots(block_table: torch.Tensor, ctx_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                 free_state: torch.Tensor, *, page_size: int, max_tokens: int, advance: bool = False) -> SlotPlan:
    """Pages and slots for new_lens[r] more tokens of each request, in one launch.

    block_table int32 [R, max_pages], R at most 16384: the entries of a
    request's new pages are written, the others left as they are.  ctx_lens int32 [R]: tokens cached so
    far.  new_lens int32 / int64 [R]; zero for a request without new tokens.
    free_pages int32 [num_pages] is a ring, one place for every page of the
    pool: with free_state = (head, count), the free pages are
    free_pages[(head + i) % num_pages] for i < count.  max_tokens bounds the
    batch's new tokens (the length of the slot map).  With ``advance`` ctx_lens
    and free_state are overwritten with the lengths and the state returned, as
    a captured step needs.

    A request's last page, begun earlier, must be its own.  Too few free pages,
    more tokens than max_tokens, a length past the table or a page id outside
    the pool set the device error word; the call then changes nothing, gives
    every token the slot -1 and returns starts of 0 and the old lengths.
    """
    _lib.require_cuda(block_table, ctx_lens, new_lens, free_pages, free_state)
    R, width, P = _check(block_table, ctx_lens, free_pages, free_state, new_lens, "new_lens", page_size)
    if new_lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"new_lens must be int32 or int64, got {new_lens.dtype}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
    new_lens = _lib.int32(new_lens)
    # one allocation: slots and positions (each at a multiple of 16 bytes), starts, and the lengths and state where
    # they are not written over
    pad = -max_tokens % 4
    sizes = [max_tokens, pad, max_tokens, pad, R + 1, R, 2] if pad else [max_tokens, max_tokens, R + 1, R, 2]
    if advance:
        sizes = sizes[:-2]
    parts = ctx_lens.new_empty(sum(sizes)).split_with_sizes(sizes)
    slots, positions, starts = (parts[0], parts[2], parts[4]) if pad else parts[:3]
    lens_out, state_out = (ctx_lens, free_state) if advance else parts[-2:]
    with _lib.device_of(ctx_lens):
        st = _lib.direct().ffa_assign_slots(
            block_table.data_ptr(), width, ctx_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(),
            free_state.data_ptr(), slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
            lens_out.data_ptr(), state_out.data_ptr(), R, P, page_size, max_tokens, _lib.err_ptr(ctx_lens),
            _lib.stream_of(ctx_lens))
    _lib.check(st, "ffa_assign_slots")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(ctx_lens.device)
    return SlotPlan(slots, positions, starts, lens_out, state_out)


def release_pages(block_table: torch.Tensor, ctx_lens: torch.Tensor, done: torch.Tensor, free_pages: torch.Tensor,
                  free_state: torch.Tensor, *, page_size: int, keep: Optional[torch.Tensor] = None,
                  advance: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Give back the pages of the requests that ``done`` [R] (bool) marks, in
    one launch: to the back of the ring, in the order of the batch and of each
    request's table.  Returns (ctx_lens, free_state) with the marked requests'
    lengths 0; block_table is left as it is.

    keep int32 [R]: the pages that hold a request's first keep[r] tokens are
    not given back (a shared prefix, which its owner gives back).  The other
    arguments as ``assign_slots``.  A length past the table, a page id outside
    the pool or more pages than the ring has places for set the device error
    word; the call then changes nothing.
    """
    _lib.require_cuda(block_table, ctx_lens, done, free_pages, free_state, keep)
    R, width, P = _check(block_table, ctx_lens, free_pages, free_state, done, "done", page_size)
    if done.dtype is not torch.bool:
        raise ValueError(f"done must be bool, got {done.dtype}")
    done = done.contiguous()
    if keep is not None:
        if keep.dtype not in (torch.int32, torch.int64) or tuple(keep.shape) != (R,):
            raise ValueError(f"keep must be int32 or int64 [{R}], got {keep.dtype} {tuple(keep.shape)}")
        keep = _lib.int32(keep)
    lens_out, state_out = (ctx_lens, free_state) if advance else ctx_lens.new_empty(R + 2).split([R, 2])
    with _lib.device_of(ctx_lens):
        st = _lib.direct().ffa_release_pages(
            block_table.data_ptr(), width, ctx_lens.data_ptr(), done.data_ptr(),
            keep.data_ptr() if keep is not None else None, free_pages.data_ptr(), free_state.data_ptr(),
            lens_out.data_ptr(), state_out.data_ptr(), R, P, page_size, _lib.err_ptr(ctx_lens),
            _lib.stream_of(ctx_lens))
    _lib.check(st, "ffa_release_pages")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(ctx_lens.device)
    return lens_out, state_out


class DevicePageTable:
    """The device tensors of one page pool: a table row and a length for each of
    ``max_requests`` requests (at most 16384), and the ring of free pages.  Every method but
    ``num_free_pages`` is one launch without a synchronisation.

    Rows are the places of a serving batch: a row of length 0 is empty.  Pass
    ``block_table`` and ``ctx_lens`` to ``paged_prefill``, ``paged_decode`` and
    ``prefix_decode``.
    """

    def __init__(self, max_requests: int, max_pages_per_request: int, num_pages: int, page_size: int = 64,
                 device: Union[torch.device, str] = "cuda"):
        if min(max_requests, max_pages_per_request, num_pages, page_size) <= 0:
            raise ValueError("DevicePageTable: sizes must be positive")
        self.page_size = page_size
        self.block_table = torch.full((max_requests, max_pages_per_request), -1, dtype=torch.int32, device=device)
        self.ctx_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.free_state = torch.tensor([0, num_pages], dtype=torch.int32, device=device)

    def assign(self, new_lens: torch.Tensor, max_tokens: int) -> SlotPlan:
        """Pages and slots for new_lens [max_requests] more tokens; the table's lengths grow by them."""
        return assign_slots(self.block_table, self.ctx_lens, new_lens, self.free_pages, self.free_state,
                            page_size=self.page_size, max_tokens=max_tokens, advance=True)

    def release(self, done: torch.Tensor, keep: Optional[torch.Tensor] = None) -> None:
        """Empty the rows that done [max_requests] marks; the pages of their first keep tokens stay taken."""
        release_pages(self.block_table, self.ctx_lens, done, self.free_pages, self.free_state,
                      page_size=self.page_size, keep=keep, advance=True)

    def share(self, owner: int, rows: Sequence[int], tokens: int) -> None:
        """Rows begin with the first ``tokens`` of row ``owner``: whole pages, which stay the owner's.  Release these
        rows with keep = tokens, and the owner after them.

        The owner has to hold that many tokens and the rows none: where they do not (a row that was released keeps
        its old entries), the device error word is set and nothing changes."""
        owner, rows, tokens = int(owner), [int(r) for r in rows], int(tokens)
        R, width, P = _check(self.block_table, self.ctx_lens, self.free_pages, self.free_state, self.ctx_lens,
                             "ctx_lens", self.page_size)
        if tokens <= 0 or tokens % self.page_size:
            raise ValueError(f"a shared prefix is whole pages of {self.page_size} tokens, got {tokens}")
        if tokens > width * self.page_size:
            raise ValueError(f"{tokens} tokens are past a row's {width} pages")
        if not 0 <= owner < R or any(not 0 <= r < R or r == owner for r in rows) or len(set(rows)) < len(rows):
            raise ValueError(f"rows must be distinct, in [0, {R}) and not the owner's")
        _lib.require_cuda(self.block_table, self.ctx_lens)
        with _lib.device_of(self.ctx_lens):
            st = _lib.load().ffa_share_pages(
                self.block_table.data_ptr(), width, self.ctx_lens.data_ptr(), owner, (ctypes.c_int * len(rows))(*rows),
                len(rows), R, P, self.page_size, tokens, _lib.err_ptr(self.ctx_lens),
                _lib.stream_of(self.ctx_lens))
        _lib.check(st, "ffa_share_pages")
        if _lib.sync_check_enabled():
            _lib.check_device_errors(self.ctx_lens.device)

    @property
    def num_free_pages(self) -> int:
        """Free pages (waits for the device)."""
        return int(self.free_state[1])
