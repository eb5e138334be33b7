"""CPU restatement, in 64 bits, of attention by formula and rules, of the paged 8-bit cache and of the page tables (test infrastructure
only).  Nothing of it has a counterpart in the reference."""
from __future__ import annotations

import math

import torch

ENTRY_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def changed_scores(q, k, pos, *, scale, softcap=None, slope=None, bias=None):
    """One head: q (n, D) at positions pos (n), k (m, D) -> scores (n, m) in float64."""
    x = scale * (q.double() @ k.double().T)
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    away = torch.arange(k.shape[0])[None, :] - pos[:, None]
    if slope is not None:
        x = x - float(slope) * away.abs()
    if bias is not None:
        radius = bias.shape[0] // 2
        x = x + bias.double()[away.clamp(-radius, radius) + radius]
    return x


def attend(x, visible, v):
    """softmax over the visible keys times v; masked places take no part, whatever they hold; rows without any give zeros."""
    out = torch.zeros(x.shape[0], v.shape[1], dtype=torch.float64)
    for i in range(x.shape[0]):
        on = visible[i]
        if bool(on.any()):
            row = x[i, on]
            if bool((row == -math.inf).all()):
                continue
            out[i] = torch.softmax(row, 0) @ v[on].double()
    return out


def visible_keys(b, q_len, k_len, *, causal=False, window=None, documents=None, prefix_lens=None, key_lens=None):
    pos = torch.arange(q_len)[:, None] + k_len - q_len
    j = torch.arange(k_len)[None, :]
    on = torch.ones(q_len, k_len, dtype=torch.bool)
    if causal:
        on &= j <= pos
    if window is not None:
        on &= (pos - j).abs() < window
    if prefix_lens is not None:
        on |= j < int(prefix_lens[b])
    if key_lens is not None:
        on &= j < int(key_lens[b])
    if documents is not None:
        on &= documents[b][None, :] == documents[b][k_len - q_len:][:, None]
    return on


def scored_attention(q, k, v, *, causal=False, window=None, softcap=None, slopes=None, distance_bias=None, documents=None, prefix_lens=None,
                     key_lens=None, softmax_scale=None):
    """float64 (B, H, Sq, D) result of `stof_b200.scored_attention` (CPU tensors)."""
    B, H, Sq, D = q.shape
    group = H // k.shape[1]
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    out = torch.empty(B, H, Sq, D, dtype=torch.float64)
    pos = torch.arange(Sq) + k.shape[2] - Sq
    for b in range(B):
        on = visible_keys(b, Sq, k.shape[2], causal=causal, window=window, documents=documents, prefix_lens=prefix_lens, key_lens=key_lens)
        for h in range(H):
            x = changed_scores(q[b, h], k[b, h // group], pos, scale=scale, softcap=softcap, slope=None if slopes is None else slopes[h],
                               bias=None if distance_bias is None else distance_bias[h])
            out[b, h] = attend(x, on, v[b, h // group])
    return out


def cache_rows(pages, scales, table_row, length, head):
    """(length, D) float64: a request's keys or values of one head."""
    size = pages.shape[2]
    rows = [pages[int(table_row[i]), head].float().double() * float(scales[int(table_row[i]), head]) for i in range(-(-length // size))]
    return torch.cat(rows)[:length] if rows else torch.zeros(0, pages.shape[3], dtype=torch.float64)


def cache_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, lengths, *, window=None, softcap=None, slopes=None, distance_bias=None,
                    softmax_scale=None):
    B, n, H, D = q.shape
    group = H // k_pages.shape[1]
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    out = torch.zeros(B, n, H, D, dtype=torch.float64)
    for b in range(B):
        length = max(int(lengths[b]), 0)
        if length == 0:
            continue
        pos = torch.arange(n) + length - n
        away = torch.arange(length)[None, :] - pos[:, None]
        on = (away <= 0) & (pos >= 0)[:, None]
        if window is not None:
            on &= away > -window
        for h in range(H):
            k = cache_rows(k_pages, k_scales, block_table[b], length, h // group)
            v = cache_rows(v_pages, v_scales, block_table[b], length, h // group)
            x = changed_scores(q[b, :, h], k, pos, scale=scale, softcap=softcap, slope=None if slopes is None else slopes[h],
                               bias=None if distance_bias is None else distance_bias[h])
            out[b, :, h] = attend(x, on, v)
    return out


def cache_append(pages, scales, x, slots):
    """Writes x (T, Hkv, D) into CPU copies of one side of a cache, in fp32 as the operator's definition has it."""
    most, size = ENTRY_MAX[pages.dtype], pages.shape[2]

    def rounded(v):
        v = v.clamp(-most, most)
        return (v.round() if pages.dtype == torch.int8 else v).to(pages.dtype)

    slots, t = slots.tolist(), 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= pages.shape[0] * size:
            t += 1
            continue
        end = t + 1
        while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % size != 0:
            end += 1
        page, row, rows = slots[t] // size, slots[t] % size, x[t:end].float()
        new = rows.abs().amax((0, 2)) * torch.tensor(1.0 / most, dtype=torch.float32)
        new = torch.where(new < torch.finfo(torch.float32).tiny, torch.zeros_like(new), new)
        if row > 0:
            old = scales[page]
            new = torch.maximum(new, old)
            for h in range(pages.shape[1]):
                if new[h] > old[h]:
                    pages[page, h, :row] = rounded(pages[page, h, :row].float() * (old[h] / new[h]))
        inv = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))
        pages[page, :, row:row + end - t] = rounded(rows * inv[None, :, None]).transpose(0, 1)
        scales[page] = new
        t = end


def page_tables(lengths, held, table, stack, count, size, new_tokens):
    """Lists in, lists out: (table, stack, slots, starts, count, missing); `table` rows and `stack` are copied."""
    table, stack = [list(r) for r in table], list(stack)
    width = len(table[0]) if table else 0
    lengths = [max(x, 0) for x in lengths]
    held = [min(max(x, 0), width * size) for x in held]
    have, need = [-(-x // size) for x in held], [-(-x // size) for x in lengths]
    give, take = sum(max(a - b, 0) for a, b in zip(have, need)), sum(max(b - a, 0) for a, b in zip(have, need))
    fresh = [max(b - a, 0) for a, b in zip(held, lengths)]
    starts = [min(sum(fresh[:i]), 2 ** 31 - 1) for i in range(len(fresh) + 1)]
    slots = [-1] * new_tokens
    count = min(max(count, 0), len(stack))
    if count + give > len(stack):
        return table, stack, slots, starts, count, len(stack) - count - give
    missing = max(take - count - give, 0) + sum(max(b - width, 0) for b in need)
    if missing > 0:
        return table, stack, slots, starts, count, min(missing, 2 ** 31 - 1)
    for r, (a, b) in enumerate(zip(have, need)):
        for i in range(b, a):
            stack[count] = table[r][i]
            count += 1
    for r, (a, b) in enumerate(zip(have, need)):
        for i in range(a, b):
            count -= 1
            table[r][i] = stack[count]
    for r in range(len(fresh)):
        for i in range(fresh[r]):
            at = held[r] + i
            if starts[r] + i < new_tokens:
                slots[starts[r] + i] = table[r][at // size] * size + at % size
    return table, stack, slots, starts, count, 0
