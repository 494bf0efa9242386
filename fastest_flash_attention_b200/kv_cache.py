"""KV caches — drop-in for the reference's ops/kv_cache.py:18-240.

``ContinuousKVCache``: contiguous [max_batch, H, max_seq, D] buffers with
per-batch lengths (kv_cache.py:18-107).

``PagedKVCache``: page pool [max_pages, H_kv, page_size, D], a FIFO free
list and per-sequence page tables with the reference's exact allocation
semantics (kv_cache.py:110-240: pages popped from the front of the free
list, freed pages appended at its back, tables grown token by token).  Slot
assignment is host bookkeeping; the K/V bytes are scattered on the device
by ``ffa_paged_append`` in one launch per call instead of a per-token loop.
Beyond the reference API, ``block_table()`` exports the tables as an int32
tensor and ``decode()`` runs the sm_100a split-KV decode directly on the
pool, with no gather.  For long conversations, sequences are forked (full
pages shared, counted), trimmed (pages that left a sliding window freed) and
compacted (first tokens and window moved to fresh pages); the bytes move in
one launch of ``copy_pages`` / ``move_tokens``.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib
from .decode import check_block_table
from .utils import check_window


class ContinuousKVCache:
    """Contiguous KV cache (kv_cache.py:18-107)."""

    def __init__(self, max_batch: int, max_seq_len: int, num_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cpu"):
        self.max_batch = max_batch
        self.max_seq_len = max_seq_len
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.k_cache = torch.zeros(max_batch, num_heads, max_seq_len, head_dim, dtype=dtype, device=device)
        self.v_cache = torch.zeros(max_batch, num_heads, max_seq_len, head_dim, dtype=dtype, device=device)
        self.seq_lens = torch.zeros(max_batch, dtype=torch.long, device=device)
        self._host_lens = [0] * max_batch

    def reset(self, batch_indices: Optional[torch.Tensor] = None):
        if batch_indices is None:
            self.seq_lens.zero_()
            self._host_lens = [0] * self.max_batch
        else:
            self.seq_lens[batch_indices] = 0
            for b in torch.as_tensor(batch_indices).flatten().tolist():
                self._host_lens[b] = 0

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Append [B, H, S_new, D] and return views [B, H, max_len, D] (kv_cache.py:68-97)."""
        B, H, S_new, D = k_new.shape
        starts = self._host_lens[:B]
        for b in range(B):
            assert starts[b] + S_new <= self.max_seq_len, \
                f"KV-cache overflow: {starts[b] + S_new} > {self.max_seq_len}"
        if all(s == starts[0] for s in starts):  # common case: one strided copy
            s0 = starts[0]
            self.k_cache[:B, :, s0:s0 + S_new] = k_new
            self.v_cache[:B, :, s0:s0 + S_new] = v_new
        else:
            for b in range(B):
                self.k_cache[b, :, starts[b]:starts[b] + S_new] = k_new[b]
                self.v_cache[b, :, starts[b]:starts[b] + S_new] = v_new[b]
        for b in range(B):
            self._host_lens[b] += S_new
        self.seq_lens[:B] += S_new
        max_len = max(self._host_lens[:B])
        return self.k_cache[:B, :, :max_len], self.v_cache[:B, :, :max_len]

    def get_cache(self, batch_size: int):
        max_len = max(self._host_lens[:batch_size]) if batch_size else 0
        if max_len == 0:
            return None, None
        return self.k_cache[:batch_size, :, :max_len], self.v_cache[:batch_size, :, :max_len]


Ids = Union[torch.Tensor, Sequence[int]]


def _id_pair(src: Ids, dst: Ids, limit: int, device: torch.device, what: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """src and dst as int32 device tensors of one length.  Ids given on the
    host are checked: each in [0, limit), destinations distinct and none of
    them a source.  Ids on the device are taken as they are (the kernels skip
    and report those outside the pool)."""
    if (isinstance(src, torch.Tensor) and isinstance(dst, torch.Tensor) and src.is_cuda
            and src.device == device == dst.device and src.dtype is torch.int32 and dst.dtype is torch.int32
            and src.dim() == dst.dim() == 1
            and src.numel() == dst.numel()):  # nothing to convert, nothing to check on the host
        return src.contiguous(), dst.contiguous()
    pair = []
    for name, ids in (("src", src), ("dst", dst)):
        t = ids if isinstance(ids, torch.Tensor) else torch.tensor(list(ids), dtype=torch.int64)
        if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be a 1-D int32 / int64 tensor or a list of {what}s")
        pair.append(t)
    if pair[0].numel() != pair[1].numel():
        raise ValueError(f"{pair[0].numel()} source and {pair[1].numel()} destination {what}s")
    if not (pair[0].is_cuda or pair[1].is_cuda):
        s, d = (t.tolist() for t in pair)
        bad = [x for x in s + d if not 0 <= x < limit]
        if bad:
            raise ValueError(f"{what} {bad[0]} is outside [0, {limit})")
        if len(set(d)) < len(d) or not set(s).isdisjoint(d):
            raise ValueError(f"destination {what}s must be distinct and none of them a source")
    if limit > 2 ** 31 - 1 and any(t.dtype is torch.int64 for t in pair):
        raise ValueError(f"{what}s are 32-bit numbers: a pool of {limit} takes int32 ones alone")
    return tuple(_lib.int32(t, limit).to(device) for t in pair)


def _check_pools(k_pages: torch.Tensor, v_pages: Optional[torch.Tensor]) -> None:
    _lib.require_cuda(k_pages, v_pages)
    if v_pages is not None and (v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype
                                or v_pages.device != k_pages.device):
        raise ValueError("k_pages and v_pages must have one shape, dtype and device")
    if not k_pages.is_contiguous() or (v_pages is not None and not v_pages.is_contiguous()):
        raise ValueError("page pools must be contiguous")


def copy_pages(k_pages: torch.Tensor, v_pages: Optional[torch.Tensor], src: Ids, dst: Ids) -> None:
    """Copy whole pages src[i] -> dst[i] inside the pools, in one launch.

    Pools [P, ...] contiguous, of any dtype whose page is an even number of
    bytes; v_pages may be None (a latent cache has one pool).  src, dst: page ids, int32 / int64 on the device (or on the
    host, where they are checked); destinations are distinct and none of them
    is a source.
    """
    _check_pools(k_pages, v_pages)
    src, dst = _id_pair(src, dst, k_pages.shape[0], k_pages.device, "page id")
    if k_pages.numel() == 0 or src.numel() == 0:
        return
    with _lib.device_of(k_pages):
        st = _lib.direct().ffa_page_copy(
            k_pages.data_ptr(), v_pages.data_ptr() if v_pages is not None else None, src.data_ptr(), dst.data_ptr(),
            src.numel(), k_pages.shape[0], k_pages.numel() // k_pages.shape[0] * k_pages.element_size(),
            _lib.err_ptr(k_pages), _lib.stream_of(k_pages))
    _lib.check(st, "ffa_page_copy")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(k_pages.device)


def move_tokens(k_pages: torch.Tensor, v_pages: Optional[torch.Tensor], src_slots: Ids, dst_slots: Ids) -> None:
    """Copy single tokens' rows (every kv head) from slot src_slots[i] to slot
    dst_slots[i] inside the pools, in one launch; slot = page * page_size +
    offset.

    Pools [P, Hkv, page_size, D], or [P, page_size, D] (a latent cache),
    contiguous, of any dtype whose row of D is an even number of bytes; v_pages
    may be None.  Slots as copy_pages' page ids.
    """
    _check_pools(k_pages, v_pages)
    if k_pages.dim() not in (3, 4):
        raise ValueError(f"pools must be [P, Hkv, page_size, D] or [P, page_size, D], got {tuple(k_pages.shape)}")
    P, page_size, D = k_pages.shape[0], k_pages.shape[-2], k_pages.shape[-1]
    src_slots, dst_slots = _id_pair(src_slots, dst_slots, P * page_size, k_pages.device, "slot")
    if k_pages.numel() == 0 or src_slots.numel() == 0:
        return
    with _lib.device_of(k_pages):
        st = _lib.direct().ffa_token_move(
            k_pages.data_ptr(), v_pages.data_ptr() if v_pages is not None else None, src_slots.data_ptr(),
            dst_slots.data_ptr(), src_slots.numel(), k_pages.shape[1] if k_pages.dim() == 4 else 1, page_size, P,
            D * k_pages.element_size(), _lib.err_ptr(k_pages), _lib.stream_of(k_pages))
    _lib.check(st, "ffa_token_move")
    if _lib.sync_check_enabled():
        _lib.check_device_errors(k_pages.device)


class PagedKVCache:
    """Paged KV cache (kv_cache.py:110-240) with device-side append and decode."""

    def __init__(self, max_pages: int = 1024, page_size: int = 64, num_heads: int = 8, head_dim: int = 64,
                 dtype: torch.dtype = torch.float16, device: torch.device | str = "cpu"):
        self.max_pages = max_pages
        self.page_size = page_size
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.k_pages = torch.zeros(max_pages, num_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v_pages = torch.zeros(max_pages, num_heads, page_size, head_dim, dtype=dtype, device=device)
        self.free_pages: List[int] = list(range(max_pages))
        self.sequences: dict = {}
        self._more_owners: Dict[int, int] = {}  # page -> sequences that share it beyond the first

    # ---- allocator (kv_cache.py:157-168) ----
    def allocate_page(self) -> int:
        if not self.free_pages:
            raise RuntimeError("PagedKVCache: out of physical pages")
        return self.free_pages.pop(0)

    def free_sequence(self, seq_id: int):
        if seq_id in self.sequences:
            for page_id in self.sequences[seq_id]["page_table"]:
                self._release(page_id)
            del self.sequences[seq_id]

    def _release(self, page_id: int) -> int:
        """One owner less; a page without owners goes to the back of the free
        list.  Returns the pages freed (an entry of -1 was freed before)."""
        if page_id < 0:
            return 0
        others = self._more_owners.get(page_id, 0)
        if others:
            if others == 1:
                del self._more_owners[page_id]
            else:
                self._more_owners[page_id] = others - 1
            return 0
        self.free_pages.append(page_id)
        return 1

    def _assign_slots(self, seq_id: int, n: int) -> List[int]:
        """Slot (page * page_size + offset) of each appended token, allocating
        pages in the order of the reference's per-token loop (kv_cache.py:192-204);
        without enough free pages nothing changes."""
        seq = self.sequences.get(seq_id) or {"page_table": [], "len": 0}
        start, end, table = seq["len"], seq["len"] + n, seq["page_table"]
        more = -(-end // self.page_size) - len(table)
        if more > len(self.free_pages):
            raise RuntimeError("PagedKVCache: out of physical pages")
        table.extend(self.allocate_page() for _ in range(more))
        seq["len"] = end
        self.sequences[seq_id] = seq
        return [table[t // self.page_size] * self.page_size + t % self.page_size for t in range(start, end)]

    def _unassign_slot(self, seq_id: int) -> None:
        """Take back the last slot that _assign_slots gave a sequence (its page too, if that began with it)."""
        seq = self.sequences[seq_id]
        seq["len"] -= 1
        if seq["len"] % self.page_size == 0:
            self.free_pages.insert(0, seq["page_table"].pop())

    def append_tokens(self, seq_id: int, k_tokens: torch.Tensor, v_tokens: torch.Tensor) -> int:
        """Append [num_heads, S_new, head_dim] K/V; returns the new length (kv_cache.py:170-206)."""
        S_new = k_tokens.size(1)
        try:  # (axes of one are repeated, as the reference's assignment does)
            k_tokens, v_tokens = (t.expand(self.num_heads, S_new, self.head_dim) for t in (k_tokens, v_tokens))
        except RuntimeError:
            raise ValueError(f"append takes k and v [{self.num_heads}, tokens, {self.head_dim}], got "
                             f"{tuple(k_tokens.shape)} and {tuple(v_tokens.shape)}") from None
        new = seq_id not in self.sequences
        slots = self._assign_slots(seq_id, S_new)
        try:
            if S_new > 0:
                self._write(slots, k_tokens, v_tokens)
        except BaseException:  # nothing is cached that was not written
            for _ in slots:
                self._unassign_slot(seq_id)
            if new:
                del self.sequences[seq_id]
            raise
        return self.sequences[seq_id]["len"]

    def _append_visible(self, seq_id: int, k_tokens: torch.Tensor, v_tokens: torch.Tensor, sliding_window: int,
                       sink_tokens: int = 0) -> int:
        """A new sequence as append_tokens and trim_sequence leave it, without
        pages for the tokens that the trim would free."""
        check_window(sliding_window, sink_tokens)
        if seq_id in self.sequences:
            raise ValueError(f"PagedKVCache: sequence {seq_id} exists already")
        n, ps = k_tokens.size(1), self.page_size
        first, last = self._outside(n, sliding_window, sink_tokens)
        if first < last:  # tokens [first * ps, last * ps) get no page
            k_tokens, v_tokens = (torch.cat([t[:, :first * ps], t[:, last * ps:]], 1) for t in (k_tokens, v_tokens))
        self.append_tokens(seq_id, k_tokens, v_tokens)
        seq = self.sequences[seq_id]
        seq["page_table"][first:first] = [-1] * (last - first)
        seq["len"] = n
        return n

    def _write(self, slots: List[int], k_tokens: torch.Tensor, v_tokens: torch.Tensor) -> None:
        if self.k_pages.is_cuda and self.k_pages.dtype in _lib.DTYPE_CODE and self.head_dim % 8 == 0:
            k_new = k_tokens.to(self.k_pages.device, self.k_pages.dtype).contiguous()
            v_new = v_tokens.to(self.v_pages.device, self.v_pages.dtype).contiguous()
            slot_t = torch.tensor(slots, dtype=torch.int32).to(self.k_pages.device)
            lib = _lib.load()
            with torch.cuda.device(self.k_pages.device):
                st = lib.ffa_paged_append(k_new.data_ptr(), v_new.data_ptr(), self.k_pages.data_ptr(),
                                          self.v_pages.data_ptr(), slot_t.data_ptr(),
                                          _lib.DTYPE_CODE[self.k_pages.dtype], len(slots), self.num_heads,
                                          self.head_dim, self.page_size, self.max_pages,
                                          _lib.i64arr(k_new.stride(0), k_new.stride(1)),
                                          _lib.stream_of(self.k_pages))
            _lib.check(st, "ffa_paged_append")
        else:
            # Host-side pool (CPU or fp32): same scatter with tensor indexing.
            slot_t = torch.tensor(slots, dtype=torch.long, device=self.k_pages.device)
            pages, offs = slot_t // self.page_size, slot_t % self.page_size
            self.k_pages[pages, :, offs, :] = k_tokens.permute(1, 0, 2).to(self.k_pages)
            self.v_pages[pages, :, offs, :] = v_tokens.permute(1, 0, 2).to(self.v_pages)

    def get_kv(self, seq_id: int) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """Contiguous [num_heads, len, head_dim] copies of a sequence (kv_cache.py:208-232)."""
        if seq_id not in self.sequences or self.sequences[seq_id]["len"] == 0:
            return None, None
        seq = self.sequences[seq_id]
        L = seq["len"]
        if min(seq["page_table"]) < 0:
            raise RuntimeError(f"PagedKVCache: pages of sequence {seq_id} left its window and were freed")
        idx = torch.tensor(seq["page_table"], dtype=torch.long, device=self.k_pages.device)
        k = self.k_pages[idx].permute(1, 0, 2, 3).reshape(self.num_heads, -1, self.head_dim)[:, :L]
        v = self.v_pages[idx].permute(1, 0, 2, 3).reshape(self.num_heads, -1, self.head_dim)[:, :L]
        return k.contiguous(), v.contiguous()

    # ---- long conversations (no reference counterpart) ----
    def position(self, seq_id: int) -> int:
        """Position of the next token: the cached tokens and those that compact_sequences dropped."""
        seq = self.sequences.get(seq_id)
        return seq["len"] + seq.get("dropped", 0) if seq else 0

    def fork_sequence(self, src_id: int, dst_id: int) -> None:
        """New sequence dst_id with the same tokens as src_id."""
        self.fork_sequences([(src_id, dst_id)])

    def fork_sequences(self, pairs: Sequence[Tuple[int, int]]) -> None:
        """New sequences with the tokens of existing ones, (source, new) for
        each.  Full pages are never written again, so they are shared and
        counted; a last page in part filled is copied, all of them in one
        launch.  A failing call changes nothing."""
        made = [d for _, d in pairs]
        for s, d in pairs:
            if s not in self.sequences:
                raise KeyError(f"PagedKVCache: no sequence {s} to fork")
            if d in self.sequences or made.count(d) > 1:
                raise ValueError(f"PagedKVCache: sequence {d} exists already")
        old = [self.sequences[s]["page_table"][-1] for s, _ in pairs if self.sequences[s]["len"] % self.page_size]
        new = self.free_pages[:len(old)]
        if len(new) < len(old):
            raise RuntimeError("PagedKVCache: out of physical pages")
        if old and self.k_pages.is_cuda:
            copy_pages(self.k_pages, self.v_pages, old, new)
        elif old:  # host-side pool
            self.k_pages[new] = self.k_pages[old]
            self.v_pages[new] = self.v_pages[old]
        for s, d in pairs:
            seq = self.sequences[s]
            table = list(seq["page_table"])
            last = [self.allocate_page()] if seq["len"] % self.page_size else []  # new's pages, in order
            if last:
                table.pop()
            for page in table:
                if page >= 0:
                    self._more_owners[page] = self._more_owners.get(page, 0) + 1
            self.sequences[d] = dict(seq, page_table=table + last)

    def _outside(self, n: int, sliding_window: int, sink_tokens: int) -> Tuple[int, int]:
        """Pages [first, last) of n tokens: those without a token of the window or of the first sink_tokens."""
        first = -(-sink_tokens // self.page_size)
        return first, max(first, (n - sliding_window) // self.page_size)

    def trim_sequence(self, seq_id: int, sliding_window: int, sink_tokens: int = 0) -> int:
        """Free the pages whose tokens are all outside the last sliding_window
        tokens and the first sink_tokens (their table entries become -1; the
        windowed decode never reads them).  Returns the pages freed."""
        check_window(sliding_window, sink_tokens)
        seq = self.sequences[seq_id]
        table, freed = seq["page_table"], 0
        for i in range(*self._outside(seq["len"], sliding_window, sink_tokens)):
            freed += self._release(table[i])
            table[i] = -1
        return freed

    def compact_sequences(self, seq_ids: Sequence[int], sliding_window: int, sink_tokens: int = 0) -> int:
        """Drop every token outside the last sliding_window and the first
        sink_tokens of each sequence and move the kept ones to fresh pages,
        densely, in one launch.  The windowed decode gives the same result
        before and after (rotated keys keep their positions; ``position()``
        goes on counting the dropped tokens).  Returns the tokens dropped; a
        failing call changes nothing."""
        check_window(sliding_window, sink_tokens)
        if len(set(seq_ids)) < len(seq_ids):
            raise ValueError("PagedKVCache: a sequence is named twice")
        ps, work = self.page_size, []
        for s in seq_ids:
            n = self.sequences[s]["len"]
            start = max(n - sliding_window, 0)
            sinks = min(sink_tokens, start)
            if sinks < start:
                work.append((s, np.r_[0:sinks, start:n]))
        src, dst, dropped = [], [], 0
        for s, kept in work:
            seq = self.sequences[s]
            old = np.asarray(seq["page_table"], dtype=np.int64)
            src.append(old[kept // ps] * ps + kept % ps)
            if src[-1].min() < 0:
                raise RuntimeError(f"PagedKVCache: pages of sequence {s} in this window were freed")
        pages = [-(-len(kept) // ps) for _, kept in work]
        if sum(pages) > len(self.free_pages):
            raise RuntimeError("PagedKVCache: out of physical pages")
        first = 0
        for (_, kept), count in zip(work, pages):
            fresh = np.asarray(self.free_pages[first:first + count], dtype=np.int64)
            at = np.arange(len(kept))
            dst.append(fresh[at // ps] * ps + at % ps)
            first += count
        if work:
            src_t, dst_t = (torch.from_numpy(np.concatenate(x)) for x in (src, dst))
            if self.k_pages.is_cuda:
                move_tokens(self.k_pages, self.v_pages, src_t.to(self.k_pages.device), dst_t)
            else:  # host-side pool
                for pool in (self.k_pages, self.v_pages):
                    pool[dst_t // ps, :, dst_t % ps] = pool[src_t // ps, :, src_t % ps]
        old = [self.sequences[s]["page_table"] for s, _ in work]
        for (s, kept), count in zip(work, pages):
            seq = self.sequences[s]
            seq["page_table"] = [self.allocate_page() for _ in range(count)]  # the fresh ones, in order
            dropped += seq["len"] - len(kept)
            seq["dropped"] = seq.get("dropped", 0) + seq["len"] - len(kept)
            seq["len"] = len(kept)
        for table in old:
            for page in table:
                self._release(page)
        return dropped

    @property
    def num_free_pages(self) -> int:
        return len(self.free_pages)

    @property
    def total_capacity(self) -> int:
        return self.max_pages * self.page_size

    # ---- device views for the decode kernel ----
    def block_table(self, seq_ids: Sequence[int], device=None, *, sliding_window: Optional[int] = None,
                    sink_tokens: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """(block_table int32 [R, max_pages_of_batch], ctx_lens int32 [R]) on
        `device`.  With a window, pages outside it may have been freed."""
        device = device or self.k_pages.device
        tables = [self.sequences[s]["page_table"] for s in seq_ids]
        width = max(1, max(len(t) for t in tables))
        bt = torch.zeros(len(seq_ids), width, dtype=torch.int32)
        for i, t in enumerate(tables):
            if t:
                bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        lens = torch.tensor([self.sequences[s]["len"] for s in seq_ids], dtype=torch.int32)
        check_block_table(bt, lens, self.max_pages, self.page_size, sliding_window, sink_tokens)
        return bt.to(device), lens.to(device)

    def decode(self, q: torch.Tensor, seq_ids: Sequence[int], *, scale: Optional[float] = None,
               softcap: Optional[float] = None, return_lse: bool = False, sliding_window: Optional[int] = None,
               sink_tokens: int = 0):
        """One-token attention of q [R, Hq, D] over each sequence's cached K/V
        (with a window: over its last tokens and the first sink_tokens)."""
        from .decode import paged_decode

        bt, lens = self.block_table(seq_ids, q.device, sliding_window=sliding_window, sink_tokens=sink_tokens)
        max_ctx = max(self.sequences[s]["len"] for s in seq_ids)
        return paged_decode(q, self.k_pages, self.v_pages, bt, lens, scale=scale, softcap=softcap,
                            return_lse=return_lse, max_ctx=max_ctx, sliding_window=sliding_window,
                            sink_tokens=sink_tokens)
