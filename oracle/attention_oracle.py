"""float64 restatement of the operators between the qkv and the output projection (include/sonar_attention.h says the formulas).
Arrays in, arrays out; nothing is rounded."""
from __future__ import annotations

import numpy as np


def qk_norm_rope(x, positions=None, table=None, weight=None, epsilon=1e-6, half=True):
    """Norm and rotation of heads x (tokens, heads, dim)."""
    y = np.array(x, dtype=np.float64)
    if weight is not None:
        with np.errstate(invalid="ignore", over="ignore"):
            y = y / np.sqrt((y * y).mean(axis=-1, keepdims=True) + epsilon) * np.asarray(weight, dtype=np.float64)
    if table is None:
        return y
    rotary = table.shape[1]
    known = (positions >= 0) & (positions < table.shape[0])
    rows = np.full((len(positions), rotary), np.nan)
    rows[known] = np.asarray(table, dtype=np.float64)[positions[known]]
    cos, sin = rows[:, None, :rotary // 2], rows[:, None, rotary // 2:]
    first = np.arange(rotary // 2) if half else np.arange(0, rotary, 2)
    second = first + (rotary // 2 if half else 1)
    a, b = y[..., first].copy(), y[..., second].copy()
    with np.errstate(invalid="ignore"):
        y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y


def append(cache, rows, slots):
    """cache (pages, page_size, heads, dim) with rows (tokens, heads, dim) at their slots."""
    out = np.array(cache, dtype=np.float64)
    pages, page_size = out.shape[:2]
    for row, slot in zip(rows, slots):
        if 0 <= slot < pages * page_size:
            out[slot // page_size, slot % page_size] = row
    return out


def visible(length, queries, causal=True, window=0, tree=None):
    """(queries, length): whether a sequence's queries see its keys; tree: their words, (queries, words)."""
    seen = np.zeros((queries, length), dtype=bool)
    for j in range(queries):
        at = length - queries + j
        for p in range(length):
            if tree is not None:
                c = p - (length - queries)
                seen[j, p] = c < 0 or (c < 64 * tree.shape[1] and (int(tree[j, c // 64]) >> (c % 64)) & 1 == 1)
            elif causal:
                seen[j, p] = p <= at and (window == 0 or p > at - window)
            else:
                seen[j, p] = True
    return seen


def paged_attention(q, k_cache, v_cache, table, lens, starts, scale, causal=True, window=0, cap=0.0, slopes=None, tree=None):
    """(out, mean of |v| with the same weights, largest |q| . |k| * scale that a query sees): the last two for tolerances."""
    q, k_cache, v_cache = (np.asarray(x, dtype=np.float64) for x in (q, k_cache, v_cache))
    tokens, heads, dim = q.shape
    page_size, kv_heads = k_cache.shape[1:3]
    out, size, most = np.zeros_like(q), np.zeros_like(q), np.zeros((tokens, heads))
    for i, length in enumerate(lens):
        length = max(0, min(int(length), table.shape[1] * page_size))
        first, queries = int(starts[i]), int(starts[i + 1] - starts[i])
        seen = visible(length, queries, causal, window, None if tree is None else tree[first:first + queries])
        needed = seen.any(axis=0)
        keys = np.arange(length)
        pages = np.where(needed, table[i][keys // page_size], 0) if length else keys
        distance = np.abs(keys[None, :] - (length - queries + np.arange(queries))[:, None])
        for h in range(heads):
            g = h // (heads // kv_heads)
            k, v = k_cache[pages, keys % page_size, g], v_cache[pages, keys % page_size, g]
            with np.errstate(all="ignore"):
                s = q[first:first + queries, h] @ k.T * scale
                bound = np.abs(q[first:first + queries, h]) @ np.abs(k).T * scale
                if cap > 0:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s - slopes[h] * distance
                for j in range(queries):
                    see = seen[j]
                    if not see.any():
                        continue
                    e = np.exp(s[j, see] - s[j, see].max())
                    out[first + j, h] = e @ v[see] / e.sum()
                    size[first + j, h] = e @ np.abs(v[see]) / e.sum()
                    most[first + j, h] = bound[j, see].max()
    return out, size, most
