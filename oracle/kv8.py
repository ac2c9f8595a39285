"""The paged INT8 KV cache operators (include/leafq.h, leafq_kv8_*) from their
definitions in 64-bit floats: what the GPU tests compare with."""
from __future__ import annotations

import numpy as np


def pages_of(n: int, page: int) -> int:
    return -(-n // page)


def plan(context, new, table, free, taken: int, page: int, tokens: int):
    """leafq_kv8_plan.  Returns a dict of its outputs; table is a copy."""
    table = np.array(table)
    rows, max_pages = table.shape
    lengths, token_offsets, page_offsets, positions, slots = [], [0], [0], [], []
    wanted, taken_after = 0, taken
    for s in range(rows):
        c, n = int(context[s]), int(new[s])
        before, after = pages_of(c, page), pages_of(c + n, page)
        fits = after <= max_pages
        need = after - before if fits else 0
        wanted += need
        granted = fits and (need == 0 or taken + wanted <= len(free))
        if granted and need:
            table[s, before:after] = free[taken + wanted - need:taken + wanted]
            taken_after = taken + wanted
        length = c + n if granted else c
        lengths.append(length)
        token_offsets.append(token_offsets[-1] + n)
        page_offsets.append(page_offsets[-1] + pages_of(length, page))
        for p in range(c, c + n):
            positions.append(p)
            slots.append(int(table[s, p // page]) * page + p % page if granted else -1)
    pad = tokens - len(positions)
    return dict(table=table, lengths=np.array(lengths), token_offsets=np.array(token_offsets),
                page_offsets=np.array(page_offsets), positions=np.array(positions + [0] * pad),
                slots=np.array(slots + [-1] * pad), taken=taken_after)


def rotate(x, positions, rope):
    """Rotates the first 2 * cos.shape[1] elements of x [tokens, heads, dim]."""
    x = np.array(x, dtype=np.float64)
    if rope is None:
        return x
    cos, sin = (np.asarray(t, dtype=np.float64)[positions][:, None] for t in rope)
    half = cos.shape[-1]
    a, b = x[..., :half].copy(), x[..., half:2 * half].copy()
    x[..., :half] = a * cos - b * sin
    x[..., half:2 * half] = b * cos + a * sin
    return x


def append(x, slots, codes, scales):
    """One of leafq_kv8_append's two sides: rows x [tokens, heads, dim]
    (rotated already) into codes [pages, heads, page, dim] (real numbers
    before rounding are returned beside them, for ties)."""
    x = np.asarray(x, dtype=np.float64)
    codes, scales = codes.astype(np.float64), scales.astype(np.float64)
    unrounded = codes.copy()
    page = codes.shape[2]
    i = 0
    while i < len(slots):
        if slots[i] < 0:
            i += 1
            continue
        p, first = divmod(int(slots[i]), page)
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and first + n < page:
            n += 1
        for h in range(codes.shape[1]):
            rows = x[i:i + n, h]
            need = max(np.abs(rows).max() / 127, 1e-12)
            scale = max(scales[p, h], need) if first else need
            if first and scale > scales[p, h]:
                unrounded[p, h, :first] = codes[p, h, :first] * (scales[p, h] / scale)
                codes[p, h, :first] = np.rint(unrounded[p, h, :first])
            unrounded[p, h, first:first + n] = rows / scale
            codes[p, h, first:first + n] = np.clip(np.rint(rows / scale), -127, 127)
            scales[p, h] = scale
        i += n
    return codes, scales, unrounded


def attention(q, visible, keys, values, scale):
    """Rows q [rows, group, dim] of one kv head over its keys and values
    [n, dim], row r seeing the first visible[r].  Returns (out, reach), reach
    the largest scale * sum |q||k| of each query: what rounding grows with."""
    out = np.zeros_like(q)
    reach = np.zeros(q.shape[:2])
    for r, n in enumerate(visible):
        if n <= 0:
            continue
        x = q[r] @ keys[:n].T * scale
        reach[r] = (np.abs(q[r]) @ np.abs(keys[:n]).T * scale).max(axis=1)
        e = np.exp(x - x.max(axis=1, keepdims=True))
        out[r] = e @ values[:n] / e.sum(axis=1, keepdims=True)
    return out, reach
