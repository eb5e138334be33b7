"""Attention whose scores are changed by a formula and masked by rules, and its form for generation token by token over a paged 8-bit
key/value cache (host side of `stof_scored_attn`, `stof_cache_attn`, `stof_cache_append` and `stof_page_tables`; argument checks and
launches are in `csrc/host/stof_native.cpp`).  Forward only, like every operator here."""
from __future__ import annotations

from . import _lib


def scored_attention(q, k, v, *, causal: bool = False, window=None, softcap=None, slopes=None, distance_bias=None, documents=None,
                     prefix_lens=None, key_lens=None, softmax_scale=None, out=None):
    """q (B, H, Sq, D), k and v (B, Hkv, Sk, D) -> (B, H, Sq, D); float16 or bfloat16, D 64 or 128, H a multiple of Hkv (query head h reads
    K/V head h // (H // Hkv)); any strides with a contiguous last dimension (others, and addresses and strides that are not multiples
    of 16 bytes, are packed first).  Query i sits at position i + Sk - Sq among the keys.

    Scores, in this order: x = softmax_scale * q.k (default 1 / sqrt(D)); `softcap`: x = softcap * tanh(x / softcap); `slopes` (H) float32:
    x -= slopes[h] * |position - j|; `distance_bias` (H, 2R + 1) float32, R at most 2048: x += distance_bias[h, R + clamp(j - position, -R, R)].
    The capped score is off by up to 7e-6 of itself.  Minus infinity in the table takes keys out; a finite low value leaves them visible, and
    a query that sees nothing else averages over them.

    Key j is visible where j < key_lens[b], documents[b, j] == documents[b, position], and either j < prefix_lens[b] or (not causal or
    j <= position) and (no window or |position - j| < window).  `key_lens`, `prefix_lens` (B) and `documents` (B, Sk; Sq <= Sk) are int32;
    a prefix needs `causal`.  A query without any visible key gives zeros.

    Keys and values at or behind key_lens[b] may hold anything.  In front of it a NaN or an infinity in v reaches every query whose
    128-key tile holds it, visible or not."""
    return (_lib._native or _lib.native()).scored_attention(q, k, v, out, causal, window, softcap, slopes, distance_bias, documents, prefix_lens,
                                                            key_lens, softmax_scale)


def cache_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, *, window=None, softcap=None, slopes=None, distance_bias=None,
                    softmax_scale=None, out=None):
    """Attention of the last n tokens of every request over a paged cache: q (B, n, H, D) -> (B, n, H, D), float16 or bfloat16.

    `k_pages`, `v_pages` (pages, Hkv, page_size, D) int8 or float8_e4m3fn, contiguous; `k_scales`, `v_scales` (pages, Hkv) float32: an entry
    stands for entry * scale.  Key j of request b lies in page block_table[b, j // page_size] (int32), row j % page_size.  Token t sits
    at position lengths[b] - n + t (`lengths` int32, the new tokens included) and sees what is not behind it and, with `window`, less
    than `window` away.  `softcap`, `slopes`, `distance_bias` and `softmax_scale` as for `scored_attention`.  Requests of length 0, and tokens at
    negative positions, give zeros.  A page number outside the cache is reported through the status word, its keys are left out and the result
    is not to be used; the table may hold anything behind a request's length and for pages that the window hides from all of its tokens.

    The weights are rounded to 16 bits relative to the largest that has entered a sum, whatever the pages' scales.  A NaN or an infinity in
    a value that one of a request's tokens sees reaches its other tokens too; one in a page's scale those that see the page."""
    return (_lib._native or _lib.native()).cache_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, out, window, softcap, slopes,
                                                           distance_bias, softmax_scale)


def cache_append(k_pages, v_pages, k_scales, v_scales, k, v, slots) -> None:
    """Writes k, v (T, Hkv, D; float16 or bfloat16, slices of a projection's rows will do) into the cache: token t into slot slots[t] =
    page * page_size + row (int32; negative: nowhere).

    Tokens of consecutive slots inside one page are a run.  A run that begins its page sets the page's scales to its largest magnitude
    per head / 127 (int8) or / 448 (e4m3), and what the page held counts no more; any other keeps the larger of that and the scale
    that is there and, where the scale grows, the entries in front of the run are rounded again to it.  entry = round(x * (1 / scale)).

    A page may hold one run of a call only: with two runs in one page - the same slot twice, say - its contents and scales are
    undefined.  Keys and values have pages and scales of their own.  Slots behind the cache are reported through the status word and
    not written.  An infinity in k or v makes its page's scale infinite, a NaN makes an int8 page's scale NaN (an e4m3 page holds it as
    an entry), until a run begins the page again."""
    (_lib._native or _lib.native()).cache_append(k_pages, v_pages, k_scales, v_scales, k, v, slots)


def page_tables(lengths, held, block_table, free_pages, free_count, page_size: int, new_tokens: int):
    """Block tables and slot map for requests that held `held` (B) tokens and shall hold `lengths` (B), all int32 on the GPU.

    `block_table` (B, W) is updated in place (entries behind a request's need stay as they are); `free_pages` is a stack of page numbers
    of which the first `free_count` (1) are on it.  Pages no longer needed are pushed, request by request and front to back; then the
    pages needed are popped in the same order.  Returns (slots, starts, free_count, missing): `slots` (new_tokens) int32, where
    slots[starts[r] + i] is the slot of token held[r] + i of request r and -1 stands behind the last; `starts` (B + 1) int32; the stack's
    new count (1); `missing` (1) = 0.

    All or nothing: where the stack has too few pages, or a row of the table too few entries, `missing` is the number of pages short, all slots
    are -1 and the table, the stack and its count stay as they were; where pages given back do not fit the stack it is negative."""
    return (_lib._native or _lib.native()).page_tables(lengths, held, block_table, free_pages, free_count, page_size, new_tokens)
