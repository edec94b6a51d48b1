"""Scaled 8-bit paged K/V cache, and the pages of a cache.

The serving cache in half the bytes of bf16: 8-bit codes (float8_e4m3fn or
int8) with one fp32 scale per (page, KV head), for K and for V.

* ``cache8_append`` quantises new tokens into their pages;
* ``cache8_attend`` attends single tokens, a few tokens per request or prompt
  rows over it: a sliding window, first tokens that stay visible (sinks), and
  the router's selected blocks with their bias (``paged.route_decode``'s
  out_idx / out_bias);
* ``pages_free``, ``pages_extend``, ``pages_fork``, ``pages_compact`` keep
  block tables and reference counts, and copy or move pages of any
  page-indexed tensors (K, V, scales, index keys, k_bar).

``Cache8`` and ``PageTable`` hold the tensors of the two for a program that
wants them kept together; every method is one of the functions.  The reference
has no counterpart (its fp8 cache has no scales, attend_triton.py:545, 626; its
pages are the serving engine's).
"""

from __future__ import annotations

import torch

from .ops import (cache8_append, cache8_attend, pages_compact, pages_extend, pages_fork,  # noqa: F401
                  pages_free)


class Cache8:
    """One layer's scaled 8-bit K/V cache.  A (page, head) tile, the unit that
    one scale covers, is one run of block_size * head_dim bytes; ``k`` and
    ``v`` are the [pages, block_size, kv heads, head_dim] views of that."""

    def __init__(self, num_pages: int, block_size: int, num_kv_heads: int, head_dim: int,
                 dtype=torch.float8_e4m3fn, device="cuda"):
        shape = (num_pages, num_kv_heads, block_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype).transpose(1, 2)
                          for _ in range(2))
        self.k_scale, self.v_scale = (torch.ones(num_pages, num_kv_heads, device=device) for _ in range(2))

    def append(self, k, v, block_table, seq_lens=None, *, cu_seqlens=None, prefix_lens=None):
        cache8_append(k, v, self.k, self.v, self.k_scale, self.v_scale, block_table, seq_lens,
                      cu_seqlens=cu_seqlens, prefix_lens=prefix_lens)

    def attend(self, q, block_table, seq_lens=None, **kw):
        return cache8_attend(q, self.k, self.v, self.k_scale, self.v_scale, block_table, seq_lens, **kw)

    def tensors(self):
        """What moves with a page."""
        return [self.k, self.v, self.k_scale, self.v_scale]


class PageTable:
    """Block tables, lengths and reference counts of ``rows`` sequences over
    ``num_pages`` pages; ``tensors`` ([num_pages, ...]) move with the pages."""

    def __init__(self, rows: int, max_blocks: int, num_pages: int, block_size: int, tensors=(), device="cuda"):
        self.block_size, self.tensors = block_size, list(tensors)
        self.block_table = torch.full((rows, max_blocks), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)

    def free(self, rows):
        pages_free(rows, self.block_table, self.seq_lens, self.refs, block_size=self.block_size)

    def extend(self, rows, new_lens):
        return pages_extend(rows, new_lens, self.block_table, self.seq_lens, self.refs, block_size=self.block_size)

    def fork(self, parents, children):
        return pages_fork(parents, children, self.block_table, self.seq_lens, self.refs, self.tensors,
                          block_size=self.block_size)

    def compact(self):
        """In place; returns the pages in use (int32 [1], on the device)."""
        return pages_compact(self.block_table, self.refs, self.tensors, out_table=self.block_table,
                             out_refs=self.refs)[2]
