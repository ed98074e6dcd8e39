"""A paged key-value cache in plain numpy, 64 bits, a sequence and a page at a time (test infrastructure only)."""
from __future__ import annotations

import numpy as np


def n_pages(tokens: int, size: int) -> int:
    return -(-tokens // size)


def page_slots(table, lengths, new_lengths, ring, state, size: int, num_tokens: int):
    """-> (table, ring, slots, starts, granted, state), copies.  Tokens are given places one after another; pages that a shrinking sequence
    gives back cannot be taken in the same call."""
    table, ring = table.copy(), ring.copy()
    P, width = len(ring), table.shape[1]
    first, count = int(state[0]), int(state[1])
    taken, back = 0, 0
    slots, starts, granted = [], [0], []
    for b, (n, m) in enumerate(zip(lengths, new_lengths)):
        n, m = int(n), int(m)
        for j in range(min(n_pages(m, size), width), n_pages(n, size)):
            ring[(first + count + back) % P] = table[b, j]
            back += 1
        end = min(n, m)
        for position in range(n, m):
            j = position // size
            if end == position and j < width:
                if position % size == 0:
                    if taken < count:
                        table[b, j] = ring[(first + taken) % P]
                        taken += 1
                        end += 1
                else:
                    end += 1
            slots.append(int(table[b, j]) * size + position % size if position < end else -1)
        starts.append(starts[-1] + max(0, m - n))
        granted.append(end)
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    return table, ring, np.array(slots, np.int64), np.array(starts, np.int32), np.array(granted, np.int32), np.array([(first + taken) % P, count - taken + back], np.int32)


def page_means(k_pages, table, lengths, new_lengths, size: int):
    """-> {page: mean [heads, d]} of the pages whose tokens change."""
    out = {}
    for b, (n, m) in enumerate(zip(lengths, new_lengths)):
        if n == m:
            continue
        for j in range(min(n, m) // size, n_pages(int(m), size)):
            page = int(table[b, j])
            if 0 <= page < len(k_pages):
                out[page] = k_pages[page, :min(size, int(m) - j * size)].astype(np.float64).mean(0)
    return out


def select_pages(q, means, table, lengths, size: int, count: int, first: int = 1, last: int = 1):
    B, heads, d = q.shape
    H = means.shape[1]
    out = np.full((B, H, count), -1, np.int32)
    for b in range(B):
        n = n_pages(int(lengths[b]), size)
        for h in range(H):
            together = q[b].reshape(H, heads // H, d)[h].astype(np.float64).sum(0)
            page = table[b, :n]
            ok = (page >= 0) & (page < len(means))
            score = np.matmul(means[np.where(ok, page, 0), h].astype(np.float64), together)
            always = [i for i in range(n) if ok[i] and (i < first or i >= n - last)]
            rest = [i for i in range(n) if ok[i] and not (i < first or i >= n - last)]
            # not a number first, then the largest, the lowest number among equals
            rest.sort(key=lambda i: (not np.isnan(score[i]), -score[i] if not np.isnan(score[i]) else 0.0, i))
            missing = [i for i in range(n) if not ok[i]]  # pages that are not in the pool, where there are no others
            pick = sorted((always + rest + missing)[:count]) if n > count else list(range(n))
            out[b, h, :len(pick)] = pick
    return out


def attention(q, k_pages, v_pages, table, lengths, scale: float, window: int = 0, slopes=None, pages=None):
    """-> (out, lse, sum of weight * |v|, largest sum of |q_i k_i|), each per (sequence, query head)."""
    B, heads, d = q.shape
    P, size, H, _ = k_pages.shape
    G = heads // H
    out, weight = np.zeros((B, heads, d)), np.zeros((B, heads, d))
    lse, spread = np.full((B, heads), -np.inf), np.zeros((B, heads))
    for b in range(B):
        n = int(lengths[b])
        for h in range(H):
            numbers = range(n_pages(n, size)) if pages is None else [j for j in pages[b, h, :n_pages(n, size)] if 0 <= j < table.shape[1]]
            ks, vs, at = [], [], []
            for j in numbers:
                page, here = int(table[b, j]), min(size, n - int(j) * size)
                low = max(0, n - window - int(j) * size) if window else 0
                if 0 <= page < P and here > low:
                    ks.append(k_pages[page, low:here, h])
                    vs.append(v_pages[page, low:here, h])
                    at.append(np.arange(low, here) + int(j) * size)
            if not ks:
                continue
            k, v, at = np.concatenate(ks).astype(np.float64), np.concatenate(vs).astype(np.float64), np.concatenate(at)
            for g in range(h * G, (h + 1) * G):
                x = q[b, g].astype(np.float64)
                s = k @ x * scale
                if slopes is not None:
                    s = s - float(slopes[g]) * (n - 1 - at)
                top = s.max()
                w = np.exp(s - top)
                lse[b, g] = top + np.log(w.sum())
                w /= w.sum()
                out[b, g], weight[b, g] = w @ v, w @ np.abs(v)
                spread[b, g] = (np.abs(k) @ np.abs(x)).max() * scale + (0 if slopes is None else float(slopes[g]) * n)
    return out, lse, weight, spread
