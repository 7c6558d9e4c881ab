"""The model step's operators on a paged cache, from their definitions, in
float64 on the host (Python integers for the tables)."""

from __future__ import annotations

import torch

PAGE = 128


def step_tables(computed, new, offsets, rows, page_tokens, num_tokens, max_blocks):
    """(query_start_loc, seq_lens, positions, slot_mapping, block_table) as lists."""
    start, lens, positions, slots, table = [0], [], [], [], []
    k = page_tokens // PAGE
    for r, row in enumerate(rows):
        fresh = min(max(new[r], 0), num_tokens - start[-1])
        length = max(computed[r] + fresh - offsets[r], 0)
        pages = [i * k + j if i >= 0 else -1 for i in row for j in range(k)][:max_blocks]
        table.append([pages[j] if j < len(pages) and j * PAGE < length else -1 for j in range(max_blocks)])
        for i in range(fresh):
            p = computed[r] + i - offsets[r]
            page = pages[p // PAGE] if p >= 0 and p // PAGE < len(pages) else -1
            positions.append(computed[r] + i)
            slots.append(page * PAGE + p % PAGE if page >= 0 else -1)
        start.append(start[-1] + fresh)
        lens.append(length)
    padding = num_tokens - start[-1]
    return start, lens, positions + [0] * padding, slots + [-1] * padding, table


def axis_of_frequency(freq, sections, order):
    if order == "blocked":
        return [axis for axis, n in enumerate(sections) for _ in range(n)]
    return [f % len(sections) if f // len(sections) < sections[f % len(sections)] else 0 for f in range(freq)]


def rotate(x, positions, omega, sections, order, style):
    """x [tokens, heads, D] rotated, float64; positions [axes, tokens]."""
    freq = omega.numel()
    out = x.double().clone()
    for f, axis in enumerate(axis_of_frequency(freq, sections, order)):
        theta = positions[axis].double() * omega[f].double()
        a, b = (f, freq + f) if style == "half" else (2 * f, 2 * f + 1)
        c, s = theta.cos()[:, None], theta.sin()[:, None]
        u, w = x[..., a].double(), x[..., b].double()
        out[..., a], out[..., b] = u * c - w * s, u * s + w * c
    return out


def attend(q, k_cache, v_cache, start, seq_lens, table, *, scale, window=0, sinks=0):
    """(out, spread, rel): the attention in float64; the same with |v|; and a
    bound on a weight's relative error from scores summed in float32 (products
    of 16-bit values are exact there): D additions of terms up to sum |q k|.
    Rows outside every request are NaN, rows that see no key zero."""
    tokens, heads, dim = q.shape
    kv = k_cache.shape[2]
    group = heads // kv
    out = torch.full((tokens, heads, dim), float("nan"), dtype=torch.float64)
    spread, rel = torch.zeros_like(out), torch.zeros(tokens, heads, 1, dtype=torch.float64)
    pages_there = k_cache.shape[0]
    for r in range(len(start) - 1):
        fresh = start[r + 1] - start[r]
        for i in range(fresh):
            p, t = seq_lens[r] - fresh + i, start[r] + i
            keys = torch.arange(min(p + 1, table.shape[1] * PAGE)) if p >= 0 else torch.arange(0)
            if window:
                keys = keys[(p - keys < window) | (keys < sinks)]
            page = table[r].long()[keys // PAGE]
            there = (page >= 0) & (page < pages_there)
            page, row = page[there], keys[there] % PAGE
            out[t] = 0
            if not len(page):
                continue
            k, v = k_cache[page, row].double(), v_cache[page, row].double()  # [keys, kv, D]
            qh = q[t].double().view(kv, group, dim)
            logits = torch.einsum("hgd,khd->hgk", qh, k) * scale
            weights = torch.softmax(logits, -1)
            out[t] = torch.einsum("hgk,khd->hgd", weights, v).reshape(heads, dim)
            spread[t] = torch.einsum("hgk,khd->hgd", weights, v.abs()).reshape(heads, dim)
            size = (torch.einsum("hgd,khd->hgk", qh.abs(), k.abs()) * abs(scale)).amax(-1)
            rel[t] = (2 * (dim + 4) * size * 2.0**-24).reshape(heads, 1) + 2.0**-20
    return out, spread, rel
