"""Oracle for a step over drafted tokens on the ragged paged cache (test infrastructure; see oracle/__init__.py): plain
NumPy in 64 bits from the operators' definitions, a sequence and a token at a time. The reference has no such step."""

from __future__ import annotations

import numpy as np


def rpa_plan_ref(ctx_lens, q_lens, page_indices, free_pages, n_free, page_size, tokens, pages_held=None, depths=None):
    """(kv_lens, cu_q_lens, positions, slots, pages_held, n_free, page_indices), the table as it is afterwards."""
    S = len(ctx_lens)
    table = np.array(page_indices, np.int64).reshape(S, -1).copy()
    pps = table.shape[1]
    stack = [int(p) for p in free_pages[: min(max(int(n_free[0]), 0), len(free_pages))]]
    missing = t = 0
    lens, held_out = [], []
    cu, positions, slots = [0], np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64)
    for s in range(S):
        ctx = max(int(ctx_lens[s]), 0)
        n = min(max(int(q_lens[s]), 0), tokens - t)
        held = -(-ctx // page_size) if pages_held is None else int(pages_held[s])
        held = min(max(held, 0), pps)
        served = 0
        for j in range(held, min(-(-(ctx + n) // page_size), pps)):
            if stack:
                table[s, j] = stack.pop()
                served += 1
            else:
                table[s, j] = -1
                missing += 1
        for i in range(n):
            place = ctx + i
            positions[t] = ctx + (i if depths is None else int(depths[t]))
            if place // page_size < pps and table[s, place // page_size] >= 0:
                slots[t] = table[s, place // page_size] * page_size + place % page_size
            t += 1
        lens.append(ctx + n)
        held_out.append(held + served)
        cu.append(t)
    return tuple(np.asarray(x, np.int32) for x in (lens, cu, positions, slots, held_out, [len(stack), missing],
                                                   table.reshape(-1)))


def norm_rope_f64(x, gamma, positions, cos_sin, eps, interleaved):
    """The normed and turned heads of x (T, H, D), and a bound of the size of what was added up for each element."""
    y = np.asarray(x).astype(np.float64)
    if gamma is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(gamma).astype(np.float64)
    size = np.abs(y)
    rot = cos_sin.shape[1]
    rows = np.asarray(cos_sin).astype(np.float64)[np.clip(positions, 0, len(cos_sin) - 1)]
    out = y.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = rows[:, None, i], rows[:, None, rot // 2 + i]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., a] * s + y[..., b] * c
        size[..., a] = size[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    return out, size


def pack_tree_mask(sees, words=None):
    """sees[i, j] (node i sees node j) as int32 words, 32 nodes each."""
    n, m = sees.shape
    words = max(1, -(-m // 32)) if words is None else words
    out = np.zeros((n, words), np.uint32)
    for i in range(n):
        for j in range(min(m, 32 * words)):
            if sees[i, j]:
                out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def tree_attention_f64(q, kv_cache, kv_lens, page_indices, cu_q_lens, tree_mask, distribution, sm_scale):
    """(the rows in float64, the mean of |v| under each row's weights: what the weights' rounding is relative to). Rows no
    sequence below distribution[0] has are q's. Positions a row does not see are left out, whatever they hold, and so are those
    whose table entry is no page of the cache."""
    pages, page_size, hkv, _, D = kv_cache.shape
    T, H, _ = q.shape
    S = len(kv_lens)
    table = np.asarray(page_indices).reshape(S, -1)
    out = np.asarray(q).astype(np.float64)
    size = np.zeros_like(out)
    group = H // hkv
    bits = np.asarray(tree_mask).view(np.uint32)
    for s in range(int(distribution[0])):
        t0, t1 = int(cu_q_lens[s]), int(cu_q_lens[s + 1])
        length = min(max(int(kv_lens[s]), 0), table.shape[1] * page_size)
        ctx = int(kv_lens[s]) - (t1 - t0)
        entry = table[s, np.arange(length) // page_size]
        paged = (entry >= 0) & (entry < pages)
        where = np.where(paged, entry, 0)
        rows = np.asarray(kv_cache)[where, np.arange(length) % page_size].astype(np.float64)  # (length, hkv, 2, D)
        for t in range(t0, t1):
            sees = [p for p in range(length) if paged[p] and (p < ctx or
                    (p - ctx < 32 * bits.shape[1] and (int(bits[t, (p - ctx) // 32]) >> ((p - ctx) % 32)) & 1))]
            if not sees:
                out[t] = 0
                continue
            for h in range(H):
                k, v = rows[sees, h // group, 0], rows[sees, h // group, 1]
                z = sm_scale * (k @ np.asarray(q[t, h]).astype(np.float64))
                w = np.exp(z - z.max())
                w /= w.sum()
                out[t, h] = w @ v
                size[t, h] = w @ np.abs(v)
    return out, size


def rpa_commit_ref(kv_cache, kv_lens, page_indices, cu_q_lens, paths, n_accepted):
    """(lengths, the cache afterwards)."""
    cache = np.array(kv_cache)
    pages, page_size = cache.shape[:2]
    S = len(kv_lens)
    table = np.asarray(page_indices).reshape(S, -1)
    lens = []

    def row(s, place):
        if place // page_size >= table.shape[1] or not 0 <= table[s, place // page_size] < pages:
            return None
        return table[s, place // page_size], place % page_size

    for s in range(S):
        n = int(cu_q_lens[s + 1]) - int(cu_q_lens[s])
        if n_accepted[s] < 0:
            lens.append(int(kv_lens[s]))
            continue
        ctx, last, kept = max(int(kv_lens[s]) - n, 0), -1, 0
        for d in range(min(int(n_accepted[s]), paths.shape[1])):
            node = int(paths[s, d])
            if node <= last or node >= n:
                break
            last, kept = node, kept + 1
            src, dst = row(s, ctx + node), row(s, ctx + d)
            if node != d and src is not None and dst is not None:
                cache[dst] = cache[src]
        lens.append(ctx + kept)
    return np.asarray(lens, np.int32), cache
