"""Attention for long conversations: rotary positions, a sliding window with the
first tokens kept visible, and a paged cache that holds the pages of both and
no others (no counterpart in the reference, whose modules have neither rotary
positions outside MLA nor a cache of their own).

``FastestFlashStreamingGQA`` trains and prefills; ``StreamingDecoder`` serves
it: every step is the three projections, one launch that rotates the new
queries and keys and writes keys and values into their pages, one launch of
the windowed decode, and the output projection.  Pages that leave the window
are freed as it goes, so the pool holds window + sinks tokens of a sequence,
rounded to pages.  What does grow with a sequence is its page table (an entry
for every page so far, until ``compact``), and with it a step's host time; and
positions are absolute, so a sequence ends at ``max_len``, the length of the
rotary tables, compacted or not.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .attention import fastest_flash_attn_forward, fastest_flash_attn_func
from .decode import paged_decode
from .kv_cache import PagedKVCache
from .modules import FastestFlashGQA, _heads, _merge
from .rotary import apply_rotary, rotary_append, rotary_tables
from .utils import check_window


class FastestFlashStreamingGQA(FastestFlashGQA):
    """Causal grouped-query attention with rotary positions over a sliding
    window and the first ``sink_tokens`` tokens.

    forward(x, start) takes x [B, S, hidden] whose first token has position
    ``start``; it is differentiable in training mode, as the other modules.
    ``rotary_dim`` (default: the head dim) values of each head turn, in pairs
    of ``rotary_layout``; ``rotary_scaling`` holds ``rotary_tables``' keyword
    arguments for contexts past the trained length.
    """

    def __init__(self, hidden_size: int, num_heads: int, num_kv_heads: int, head_dim: Optional[int] = None, *,
                 sliding_window: int, sink_tokens: int = 4, rotary_dim: Optional[int] = None,
                 rotary_base: float = 10000.0, rotary_layout: str = "half", rotary_scaling: Optional[dict] = None,
                 max_len: int = 32768, bias: bool = False, softcap: Optional[float] = None):
        check_window(sliding_window, sink_tokens)
        super().__init__(hidden_size, num_heads, num_kv_heads, head_dim, bias=bias, causal=True, softcap=softcap,
                         sliding_window=sliding_window, sink_tokens=sink_tokens)
        self.rotary_dim = rotary_dim or self.head_dim
        self.rotary_base = rotary_base
        self.rotary_layout = rotary_layout
        self.rotary_scaling = dict(rotary_scaling or {})
        self.max_len = max_len
        # fp32 whatever the parameters' dtype, so no buffers (which .to(dtype) would round)
        self._tables: Dict[torch.device, Tuple[torch.Tensor, torch.Tensor]] = {}

    def tables(self, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rotary tables on `device`, built at their first use."""
        if device not in self._tables:
            with torch.inference_mode(False):  # a training step may save them for its backward later
                self._tables[device] = rotary_tables(self.rotary_dim, self.max_len, self.rotary_base, device=device,
                                                     **self.rotary_scaling)
        return self._tables[device]

    def qkv(self, x: torch.Tensor, start: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q and k rotated, and v, as [B, heads, S, head_dim]."""
        B, S, _ = x.shape
        D = self.head_dim
        q = _heads(self.q_proj(x), B, S, self.num_heads, D)
        k = _heads(self.k_proj(x), B, S, self.num_kv_heads, D)
        v = _heads(self.v_proj(x), B, S, self.num_kv_heads, D)
        q, k = apply_rotary(q, k, *self.tables(x.device), start, layout=self.rotary_layout)
        return q, k, v

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """[B, S, hidden] from the rotated heads."""
        kw = dict(scale=self.scale, causal=True, softcap=self.softcap, sliding_window=self.sliding_window,
                  sink_tokens=self.sink_tokens)
        out = fastest_flash_attn_func(q, k, v, **kw) if self.training else fastest_flash_attn_forward(q, k, v, **kw)[0]
        return self.o_proj(_merge(out, q.shape[0], q.shape[2]))

    def forward(self, x: torch.Tensor, start: int = 0) -> torch.Tensor:
        return self.attend(*self.qkv(x, start))


class StreamingDecoder:
    """Prefill, decoding and forks of sequences over a FastestFlashStreamingGQA
    (fp16 or bf16 parameters on a CUDA device)."""

    def __init__(self, attn: FastestFlashStreamingGQA, max_pages: int, page_size: int = 64):
        self.attn = attn
        w = attn.q_proj.weight
        self.cache = PagedKVCache(max_pages, page_size, attn.num_kv_heads, attn.head_dim, w.dtype, w.device)

    @staticmethod
    def _check_ids(x: torch.Tensor, seq_ids: Sequence[int]) -> None:
        if len(seq_ids) != x.shape[0] or len(seq_ids) == 0:
            raise ValueError(f"{x.shape[0]} rows and {len(seq_ids)} sequences")
        if len(set(seq_ids)) < len(seq_ids):
            raise ValueError("a sequence is named twice")

    def _trim(self, seq_ids: Sequence[int]) -> None:
        for s in seq_ids:
            self.cache.trim_sequence(s, self.attn.sliding_window, self.attn.sink_tokens)

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, seq_ids: Sequence[int]) -> torch.Tensor:
        """Run new sequences' prompts x [B, S, hidden] and cache their keys and
        values (in pages for the window and the first tokens alone).  A failing
        call changes nothing."""
        m, cache = self.attn, self.cache
        self._check_ids(x, seq_ids)
        for s in seq_ids:
            if s in cache.sequences:
                raise ValueError(f"sequence {s} has a context already")
        B, S, _ = x.shape
        if S > m.max_len:
            raise ValueError(f"{S} tokens are past the rotary tables' {m.max_len}")
        first, last = cache._outside(S, m.sliding_window, m.sink_tokens)
        if B * (-(-S // cache.page_size) - (last - first)) > cache.num_free_pages:
            raise RuntimeError("PagedKVCache: out of physical pages")
        q, k, v = m.qkv(x)
        out = m.attend(q, k, v)
        for b, s in enumerate(seq_ids):
            cache._append_visible(s, k[b], v[b], m.sliding_window, m.sink_tokens)
        return out

    @torch.no_grad()
    def step(self, x: torch.Tensor, seq_ids: Sequence[int]) -> torch.Tensor:
        """One new token for each sequence: x [R, 1, hidden] -> [R, 1, hidden].
        A failing call changes nothing."""
        m, cache = self.attn, self.cache
        if x.dim() != 3 or x.shape[1] != 1:
            raise ValueError(f"a step takes x [R, 1, hidden], got {tuple(x.shape)}")
        self._check_ids(x, seq_ids)
        pos: List[int] = [cache.position(s) for s in seq_ids]
        if max(pos) >= m.max_len:
            raise ValueError(f"position {max(pos)} is past the rotary tables' {m.max_len}")
        starts = sum(cache.sequences.get(s, {"len": 0})["len"] % cache.page_size == 0 for s in seq_ids)
        if starts > cache.num_free_pages:  # before anything changes
            raise RuntimeError("PagedKVCache: out of physical pages")
        new = [s for s in seq_ids if s not in cache.sequences]
        slots = [cache._assign_slots(s, 1)[0] for s in seq_ids]
        try:
            out = self._step(x, seq_ids, pos, slots)
        except BaseException:
            for s in reversed(seq_ids):
                cache._unassign_slot(s)
            for s in new:
                del cache.sequences[s]
            raise
        self._trim(seq_ids)
        return out

    def _step(self, x: torch.Tensor, seq_ids: Sequence[int], pos: List[int], slots: List[int]) -> torch.Tensor:
        m, cache = self.attn, self.cache
        R, dev = x.shape[0], x.device
        H, Hkv, D = m.num_heads, m.num_kv_heads, m.head_dim
        meta = torch.tensor([pos, slots], dtype=torch.int32).to(dev, non_blocking=True)
        bt, lens = cache.block_table(seq_ids, dev, sliding_window=m.sliding_window, sink_tokens=m.sink_tokens)
        x = x[:, 0]
        q = rotary_append(m.q_proj(x).view(R, H, D), m.k_proj(x).view(R, Hkv, D), m.v_proj(x).view(R, Hkv, D),
                          *m.tables(dev), meta[0], meta[1], cache.k_pages, cache.v_pages, layout=m.rotary_layout)
        o = paged_decode(q, cache.k_pages, cache.v_pages, bt, lens, scale=m.scale, softcap=m.softcap,
                         sliding_window=m.sliding_window, sink_tokens=m.sink_tokens,
                         max_ctx=max(cache.sequences[s]["len"] for s in seq_ids))
        return m.o_proj(o.view(R, 1, H * D))

    def fork(self, pairs: Sequence[Tuple[int, int]]) -> None:
        """New sequences that continue existing ones, (source, new) for each."""
        self.cache.fork_sequences(pairs)

    def compact(self, seq_ids: Sequence[int]) -> int:
        """Move the sequences' visible tokens to fresh pages, densely; returns the tokens dropped."""
        return self.cache.compact_sequences(seq_ids, self.attn.sliding_window, self.attn.sink_tokens)

    def free(self, seq_id: int) -> None:
        self.cache.free_sequence(seq_id)
