"""Keys and values of requests that are being generated, in 8-bit pages (`GenerationCache`), for the stacks' `prefill` and `step`."""
from __future__ import annotations

import torch

from . import _lib
from .scored import cache_append, cache_attention, page_tables


class GenerationCache:
    """Paged 8-bit keys and values of up to `max_requests` requests of up to `max_length` tokens, for all layers of a stack.

    Everything lives on the GPU, the requests' lengths and the stack of free pages too: `resize` needs no host read, and a stack's
    `step` can be captured into a CUDA graph.  `pages` defaults to what all requests at their longest need.  `entries` is
    torch.int8 or torch.float8_e4m3fn."""

    def __init__(self, layers: int, heads: int, max_requests: int, max_length: int, pages=None, page_size: int = 32, head_dim: int = 64,
                 entries=torch.float8_e4m3fn, device="cuda"):
        if entries not in (torch.int8, torch.float8_e4m3fn):
            raise _lib.StofError(f"GenerationCache: entries must be int8 or float8_e4m3fn, got {entries}")
        if page_size not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise _lib.StofError("GenerationCache: page_size must be 16, 32, 64 or 128, head_dim 64 or 128")
        width = -(-int(max_length) // page_size)
        pages = int(max_requests) * width if pages is None else int(pages)
        shape = (layers, pages, heads, page_size, head_dim)
        self.page_size, self.heads, self.head_dim = page_size, heads, head_dim
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=torch.int8, device=device).view(entries) for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(shape[:3], device=device) for _ in range(2))
        self.block_table = torch.zeros(max_requests, width, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.missing = torch.zeros(1, dtype=torch.int32, device=device)
        self.refused = torch.zeros(1, dtype=torch.int32, device=device)

    @property
    def layers(self) -> int:
        return self.k_pages.shape[0]

    def resize(self, lengths, new_tokens: int):
        """Every request r is to hold lengths[r] tokens (0: it is done, and its pages are free again).  Returns (slots, starts) of
        the `new_tokens` tokens that come in, request by request.  Where pages are missing nothing changes and all slots are -1;
        `check()` tells.  Negative lengths count as 0."""
        return self._resize(lengths.clamp(min=0), new_tokens)

    def _resize(self, lengths, new_tokens: int):
        slots, starts, left, missing = page_tables(lengths, self.lengths, self.block_table, self.free_pages, self.free_count, self.page_size, new_tokens)
        self.free_count.copy_(left)
        self.lengths.copy_(torch.where(missing == 0, lengths, self.lengths))
        self.missing += missing.abs()
        return slots, starts

    def check(self):
        """Host-side check (synchronises): every `resize` so far found its pages, every `prefill` had lengths that it can serve."""
        n, refused = torch.cat((self.missing, self.refused)).tolist()
        self.missing.zero_()
        self.refused.zero_()
        if refused != 0:
            raise _lib.StofError(f"GenerationCache: {refused} calls of prefill changed nothing: they gave tokens to requests that hold some already, or "
                                 "more tokens to the requests than they brought")
        if n != 0:
            raise _lib.StofError(f"GenerationCache: {n} pages short, the last resizes changed nothing")

    def append(self, layer: int, k, v, slots):
        """Writes k, v (T, heads, head_dim) of new tokens into their slots."""
        cache_append(self.k_pages[layer], self.v_pages[layer], self.k_scales[layer], self.v_scales[layer], k, v, slots)

    def attention(self, layer: int, q, **rules):
        """q (max_requests, n, heads, head_dim) of the requests' last n tokens (`cache_attention`)."""
        return cache_attention(q, self.k_pages[layer], self.v_pages[layer], self.k_scales[layer], self.v_scales[layer], self.block_table, self.lengths,
                               **rules)
