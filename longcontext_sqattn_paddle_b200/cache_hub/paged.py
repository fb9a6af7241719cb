"""A KV cache in pages, in 16 bits or quantised to 8 or 4 as it is written, with the methods that the layer loops call
(``flash_attn_cache`` keeps one block of ``max_length`` tokens per sequence and layer; the reference has no other).

All layers share one block table: page ``i`` of a sequence is the same page of every layer's pool.  Lengths and the table
live on the GPU, so a captured decode step follows them; the host keeps copies for its own bookkeeping."""
from __future__ import annotations

from typing import List, Optional

import torch

from .. import ops


class PageAllocator:
    """Which page holds which tokens, on the host: pages are handed out from a free list and come back with ``release``."""

    def __init__(self, num_pages: int, page_size: int, batch_size: int, max_pages: int):
        self.page_size, self.max_pages = page_size, max_pages
        self.free = list(range(num_pages - 1, -1, -1))
        self.pages: List[List[int]] = [[] for _ in range(batch_size)]

    def reserve(self, b: int, tokens: int) -> List[int]:
        """Pages that sequence b gets so that it has room for ``tokens``; nothing changes where there are too few."""
        need = (int(tokens) + self.page_size - 1) // self.page_size
        if need > self.max_pages:
            raise ValueError(f"{tokens} tokens need {need} pages, the block table has {self.max_pages} a sequence")
        more = need - len(self.pages[b])
        if more > len(self.free):
            raise RuntimeError(f"the page pool is exhausted: sequence {b} needs {more} more pages, {len(self.free)} are free")
        new = [self.free.pop() for _ in range(max(0, more))]
        self.pages[b] += new
        return new

    def release(self, b: int) -> int:
        """Give back the pages of sequence b; their number."""
        n = len(self.pages[b])
        self.free += reversed(self.pages[b])
        self.pages[b] = []
        return n


class PagedKVCache:
    """``flash_attn_cache``'s methods over pages.

    A sequence of the batch begins with its prefill (or, after ``release``, with the next step's token) and takes part in every
    decode step until ``end``: from then on steps leave it out, it holds no pages and its attention is zeros.
    ``kv_format``: "native" (the 16-bit type), "int8" or "int4" (one scale per token and KV head).  ``num_pages``: size of the pool
    (default: enough for every sequence to reach ``max_length``).  ``select_pages``: a decode step attends to so many pages per
    KV head, the first ``sink_pages``, the last ``recent_pages`` and the best scoring ones; None: to all of them."""

    allocated = True

    def __init__(self, valid_start, layer_num, batch_size, max_length, num_key_value_heads, num_heads, head_dim, dtype, *,
                 kv_format: str = "int8", page_size: int = 64, num_pages: Optional[int] = None, select_pages: Optional[int] = None,
                 sink_pages: int = 1, recent_pages: int = 2, device="cuda"):
        self.valid_start, self.layer_num, self.batch_size, self.max_length = valid_start, layer_num, batch_size, max_length
        self.kv_head, self.num_heads, self.head_dim, self.dtype = num_key_value_heads, num_heads, head_dim, dtype
        self.kv_format, self.page_size, self.device = kv_format, page_size, torch.device(device)
        self.select_pages, self.sink_pages, self.recent_pages = select_pages, sink_pages, recent_pages
        if select_pages is not None and select_pages < max(1, sink_pages + recent_pages):
            raise ValueError(f"select_pages {select_pages} must hold the first {sink_pages} and the last {recent_pages} pages")
        max_pages = (max_length + page_size - 1) // page_size
        num_pages = batch_size * max_pages if num_pages is None else num_pages
        self.allocator = PageAllocator(num_pages, page_size, batch_size, max_pages)
        self.pools = [ops.PagedPool.allocate(num_pages, page_size, num_key_value_heads, head_dim, dtype, kv_format,
                                             bounds=select_pages is not None, device=self.device) for _ in range(layer_num)]
        self.block_table = torch.full((batch_size, max_pages), -1, dtype=torch.int32, device=self.device)
        self.valid_length = torch.zeros(batch_size, dtype=torch.int32, device=self.device)   # cached tokens
        self.valid_length_host = [0] * batch_size
        self.after = torch.zeros_like(self.valid_length)    # with the token of the step under way
        self.at = torch.zeros_like(self.valid_length)       # where that token goes, -1 for a sequence that has ended
        self.active = torch.ones_like(self.valid_length)    # 0: ended
        self.active_host = [True] * batch_size
        self._zero = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.context = 0

    # ---- pages ---------------------------------------------------------------------------------------------------
    def reserve(self, b: int, tokens: int) -> None:
        """Room for ``tokens`` tokens of sequence b."""
        have = len(self.allocator.pages[b])
        new = self.allocator.reserve(b, tokens)
        if new:
            self.block_table[b, have:have + len(new)] = torch.tensor(new, dtype=torch.int32).to(self.device)

    def reserve_step(self) -> None:
        """Room for the next token of every sequence that has not ended; before the replay of a captured step, which reads the table
        on the device but takes no pages of its own."""
        for b, n in enumerate(self.valid_length_host):
            if self.active_host[b]:
                self.reserve(b, n + 1)

    def bounds(self):
        """Copies of the pages' key bounds, for ``restore_bounds`` after steps that are taken back: a row that is written again
        leaves its page's bounds as wide as they were."""
        return [None if p.k_bounds is None else p.k_bounds.clone() for p in self.pools]

    def restore_bounds(self, saved) -> None:
        for pool, b in zip(self.pools, saved):
            if b is not None:
                pool.k_bounds.copy_(b)

    def release(self, b: int) -> None:
        """The pages of sequence b are free for others, and the next step's token is its first again (``end``: there is none)."""
        self.allocator.release(b)
        self.block_table[b].fill_(-1)
        self.valid_length[b] = 0
        self.valid_length_host[b] = 0

    def end(self, b: int) -> None:
        """Sequence b has ended: its pages are free for others, and decode steps, captured ones too, leave it out until a prefill
        begins another one in its place."""
        self.release(b)
        self.active[b] = 0
        self.active_host[b] = False

    # ---- the layer loops' calls ----------------------------------------------------------------------------------
    def prefill_update_kv_cache(self, query_states, key_states, value_states, layer_idx, start_bdx):
        """Write the valid part of one sequence's K/V into its pages from the first on, on the current stream."""
        bsz, seq_len, _, _ = key_states.shape
        assert bsz == 1, "Multi-batch prefilling only support prefill single batch one by one."
        assert seq_len <= self.max_length, f"Prefilling sequence length {seq_len} exceeds max length {self.max_length}."
        vs = int(self.valid_start[start_bdx] if isinstance(self.valid_start, (tuple, list)) else self.valid_start)
        valid = seq_len - vs
        if layer_idx == 0:
            self.reserve(start_bdx, valid)
            self.valid_length[start_bdx] = valid
            self.valid_length_host[start_bdx] = valid
            if not self.active_host[start_bdx]:
                self.active[start_bdx] = 1
                self.active_host[start_bdx] = True
        key, value = key_states[:, vs:], value_states[:, vs:]
        ops.paged_write(self.pools[layer_idx], key.to(self.dtype), value.to(self.dtype), self.block_table[start_bdx:start_bdx + 1], self._zero)
        if layer_idx == self.layer_num - 1 and start_bdx + bsz == self.batch_size:
            self.context += seq_len
        return key, value

    def sync(self, layer_idx, start_bdx=0):
        """Nothing to wait for: pages are written on the stream that reads them."""

    def move_gpu(self):
        """The pages are on the GPU already."""

    def decode_update_kv_cache(self, key_states, value_states, layer_idx):
        """Append one token per sequence that has not ended; ``decode_attention`` of this layer sees it."""
        if layer_idx == 0:
            if not torch.cuda.is_current_stream_capturing():
                self.reserve_step()
            torch.add(self.valid_length, self.active, out=self.after)
            torch.sub(self.after, 1, out=self.at)       # (an ended sequence has length 0)
        ops.paged_write(self.pools[layer_idx], key_states.to(self.dtype), value_states.to(self.dtype), self.block_table, self.at)
        if layer_idx == self.layer_num - 1:
            self.valid_length.copy_(self.after)
            self.count_step()

    def count_step(self) -> None:
        """The host's side of a step that has been appended."""
        self.context += 1
        self.valid_length_host = [n + int(a) for n, a in zip(self.valid_length_host, self.active_host)]

    def decode_attention(self, query, layer_idx, out_dtype=None):
        """query [B, 1, Hq, D] against the layer's pages, the step's own token among them -> [B, 1, Hq, D]."""
        pool = self.pools[layer_idx]
        if self.select_pages is not None:
            pages = ops.paged_select(query, pool, self.block_table, self.after, self.select_pages, sink_pages=self.sink_pages,
                                     recent_pages=self.recent_pages)
            return ops.paged_decode(query, pool, self.block_table, self.after, pages=pages, out_dtype=out_dtype)
        # the lengths that a captured launch will see are not known here; elsewhere a bound that changes now and then, not with every token
        bound = 0 if torch.cuda.is_current_stream_capturing() else -(-(max(self.valid_length_host) + 1) // 512) * 512
        return ops.paged_decode(query, pool, self.block_table, self.after, max_kv_len=bound, out_dtype=out_dtype)

    def read(self, layer_idx, b: int, start: int = 0, num_tokens: Optional[int] = None):
        """Keys and values [1, tokens, Hkv, D] of one sequence as they are cached, for a caller whose own prefill continues it (the rows
        of that go behind them by ``reserve`` and ``ops.paged_write``; ``prefill_update_kv_cache`` begins a sequence anew)."""
        n = self.valid_length_host[b] - start if num_tokens is None else num_tokens
        starts = torch.full((1,), start, dtype=torch.int32, device=self.device)
        return ops.paged_read(self.pools[layer_idx], self.block_table[b:b + 1], starts, n, self.valid_length[b:b + 1])
