"""Oracle of the decode step around the experts.  TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

Page plan, query/key preparation, attention over a paged cache and log probabilities, straight from their definitions in
Python integers and float64 numpy, one request and one head at a time.
"""
from __future__ import annotations

import numpy as np

LENGTH, NO_PAGE = 32, 64


def plan_pages(context, new, table, free_pages, free_count, page_size, tokens):
    """-> (starts, requests, positions, slots, lens, free_count, table, status); `table` is a new array."""
    table = np.array(table, dtype=np.int64)
    width = table.shape[1]
    count = min(max(int(free_count), 0), len(free_pages))
    status = LENGTH if count != int(free_count) else 0
    starts, requests, positions, slots, lens = [0], [], [], [], []
    left = count
    for r, (c, n) in enumerate(zip(map(int, context), map(int, new))):
        if c < 0 or n < 0:
            status |= LENGTH
            c, n = max(c, 0), max(n, 0)
        kept = min(n, tokens - len(requests))
        if kept < n or c + kept > width * page_size:
            status |= LENGTH
        for j in range(-(-c // page_size), min(-(-(c + kept) // page_size), width)):
            if left > 0:
                left -= 1
                table[r, j] = free_pages[left]
            else:
                status |= NO_PAGE
                table[r, j] = -1
        for pos in range(c, c + kept):
            j = pos // page_size
            page = int(table[r, j]) if j < width else -1
            requests.append(r), positions.append(pos), slots.append(page * page_size + pos % page_size if page >= 0 else -1)
        starts.append(len(requests)), lens.append(c + kept)
    pad = tokens - len(requests)
    return starts, requests + [-1] * pad, positions + [0] * pad, slots + [-1] * pad, lens, left, table, status


def rms_norm(x, weight, eps):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    return y if weight is None else y * np.asarray(weight, np.float64)


def rotate(x, positions, inv_freq, interleaved=False, magnitude=1.0):
    """x [tokens, heads, dim]; pairs (i, i + r/2) or (2i, 2i + 1) of the first r = 2 * len(inv_freq) elements."""
    x = np.array(x, np.float64)
    half = len(inv_freq)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    u, v = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x


def attend(q, keys, values, scale, softcap=0.0):
    """One head: q [dim], keys and values [n, dim] (the visible ones) -> (out [dim], lse, spread [dim], reach, floor [dim]) with
    what error bounds need: spread = sum p |v| / sum p, reach = largest |scale| * sum |q_i k_i|, floor = sum |v| / sum p for
    p relative to the largest."""
    q, keys, values = (np.asarray(t, np.float64) for t in (q, keys, values))
    zero = np.zeros(values.shape[1])
    if not len(keys):
        return zero, -np.inf, zero, 0.0, zero
    s = keys @ q * scale
    if softcap:
        s = softcap * np.tanh(s / softcap)
    m = s.max()
    if m == -np.inf:
        return zero, -np.inf, zero, 0.0, zero
    p = np.exp(s - m)
    return (p @ values / p.sum(), m + np.log(p.sum()), p @ np.abs(values) / p.sum(), abs(scale) * (np.abs(keys) @ np.abs(q)).max(),
            np.abs(values).sum(0) / p.sum())


def paged_attention(q, keys, values, table, lens, page_size, scale, window=0, softcap=0.0):
    """q [requests, heads, dim]; keys, values float64 [pages, kv_heads, page_size, dim] -> (out, lse, spread, reach, floor) as
    `attend`, per request and head.  A page outside the cache hides its tokens; a length past the table is cut to it."""
    q = np.asarray(q, np.float64)
    pages, kv_heads = keys.shape[:2]
    group = q.shape[1] // kv_heads
    out, lse, spread, reach, floor = np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
    for r in range(q.shape[0]):
        n = min(max(int(lens[r]), 0), table.shape[1] * page_size)
        j = np.arange(max(0, n - window) if window else 0, n)
        p, o = np.asarray(table[r])[j // page_size], j % page_size
        live = (p >= 0) & (p < pages)
        p, o = p[live], o[live]
        for g in range(kv_heads):
            k, v = keys[p, g, o], values[p, g, o]
            for h in range(g * group, (g + 1) * group):
                out[r, h], lse[r, h], spread[r, h], reach[r, h], floor[r, h] = attend(q[r, h], k, v, scale, softcap)
    return out, lse, spread, reach, floor


def token_logprobs(logits, tokens, top):
    """-> (logprobs, entropy, ids, top logprobs) of one row at a time; a row of -inf alone: -inf, 0."""
    x = np.asarray(logits, np.float64)
    rows, vocab = x.shape
    logp, ent, ids, best = np.zeros(rows), np.zeros(rows), np.full((rows, top), -1), np.full((rows, top), -np.inf)
    for r in range(rows):
        m = x[r].max()
        if np.isnan(m):
            lp = np.full(vocab, np.nan)
        elif m == -np.inf:
            lp = np.full(vocab, -np.inf)
        else:
            lp = (x[r] - m) - np.log(np.exp(x[r] - m).sum())  # m apart: a mask value of 10^38 swallows the sum
        p = np.exp(lp)
        ent[r] = -np.sum(np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0)) if not np.isnan(m) else np.nan
        t = int(tokens[r])
        logp[r] = lp[t] if 0 <= t < vocab else 0.0
        order = [int(i) for i in np.argsort(-x[r], kind="stable") if not np.isnan(x[r, i])][:top]
        ids[r, :len(order)], best[r, :len(order)] = order, lp[order]
    return logp, ent, ids, best
