"""A step with several new tokens per sequence over the paged INT8 cache, in
NumPy and 64 bits (test oracle only). One sequence, token and page at a time,
straight from the definitions of ``include/q6moe.h``.
"""

import numpy as np

from . import kv


def plan(table, lengths, counts, free_pages, free_count, page, rows, parents=None, max_count=None):
    """(starts, slots, positions, masks as sets of indices, missing, table, free_count)."""
    table = np.array(table, np.int64)
    have = max(0, min(int(free_count), len(free_pages)))
    starts, slots, positions, sees, missing = [0], [], [], [], 0
    for b in range(len(lengths)):
        n, asked = max(0, int(lengths[b])), max(0, int(counts[b]))
        c = min(asked, rows if max_count is None else max_count, rows - starts[-1])
        missing += asked - c
        if c:
            for e in range(n // page, min(table.shape[1], -(-(n + c) // page))):
                if table[b, e] < 0 and have > 0:
                    have -= 1
                    table[b, e] = free_pages[have]
        first = starts[-1]
        seen, depth = [], []
        for j in range(c):
            e = (n + j) // page
            ok = e < table.shape[1] and table[b, e] >= 0
            slots.append(int(table[b, e]) * page + (n + j) % page if ok else -1)
            missing += not ok
            if parents is None:
                positions.append(n + j)
                sees.append(None)
                continue
            p = int(parents[first + j])
            up = 0 <= p < j
            seen.append({j} | (seen[p] if up else set()))
            depth.append(depth[p] + 1 if up else 0)
            positions.append(n + depth[j])
            sees.append(seen[j])
        starts.append(first + c)
    behind = rows - len(slots)
    return (np.array(starts), np.array(slots + [-1] * behind, np.int64), np.array(positions + [0] * behind),
            sees + [set()] * behind, missing, table, have)


def masks_of(sees, words):
    """Sets of indices as int64 words."""
    out = np.zeros((len(sees), words), np.uint64)
    for i, s in enumerate(sees):
        for j in s:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def release(table, lengths, free_pages, free_count, page):
    """(table, free_pages, free_count) with every page past the cached tokens given back."""
    table, free = np.array(table), np.array(free_pages)
    have = max(0, min(int(free_count), len(free)))
    back = [(b, e) for b in range(table.shape[0]) for e in range(-(-max(0, int(lengths[b])) // page), table.shape[1])
            if table[b, e] >= 0]
    for i, (b, e) in enumerate(back):
        at = have + len(back) - 1 - i
        if at < len(free):
            free[at] = table[b, e]
            table[b, e] = -1
    return table, free, min(have + len(back), len(free))


def write(codes, scales, x, slots, group, scale_dtype):
    """Pool rows [R, C] and their scales [R, C // group] after x [rows, C] went to its slots."""
    codes, scales = np.array(codes), np.array(scales)
    new, sc = kv.quantize(x, group, scale_dtype)
    for r, s in enumerate(slots):
        if 0 <= s < codes.shape[0]:
            codes[s], scales[s] = new[r], sc[r]
    return codes, scales


def keep(pool, table, lengths, path, accepted, page):
    """Pool [pages, P, ...] after the accepted rows moved to the front."""
    old, new = np.array(pool), np.array(pool)
    pages, cap = old.shape[0], table.shape[1] * page
    for b in range(table.shape[0]):
        n = max(0, int(lengths[b]))
        for i in range(min(int(accepted[b]), path.shape[1])):
            to, at = n + i, n + path[b, i]
            if path[b, i] < 0 or max(to, at) >= cap:
                continue
            pt, pa = table[b, to // page], table[b, at // page]
            if 0 <= pt < pages and 0 <= pa < pages:
                new[pt, to % page] = old[pa, at % page]
    return new


def attention(q, k_codes, k_scales, v_codes, v_scales, table, lengths, starts, sees, page, max_count):
    """Rows of FP64 (out, spread, slope) [rows, Hq, D]; NaN where a row is left as it was.

    codes [pages, P, KVH, D], scales [pages, P, KVH]; ``sees`` a list of sets of
    new-token indices, or None for jj <= j. ``spread`` is sum p |v| / sum p, by
    which errors of the probabilities reach the output, and ``slope`` [rows, Hq]
    the largest sum |k| / sqrt(D) of a seen key, by which errors of q reach a score.
    """
    rows, hq, dim = q.shape
    kvh = k_codes.shape[2]
    out = np.full((rows, hq, dim), np.nan)
    spread, slope = np.zeros((rows, hq, dim)), np.zeros((rows, hq))
    cap = table.shape[1] * page

    def values(codes, scales, b, tokens):
        pg = table[b, tokens // page]
        ok = (pg >= 0) & (pg < codes.shape[0])
        pg = np.where(ok, pg, 0)
        v = codes[pg, tokens % page].astype(np.float64) * scales[pg, tokens % page].astype(np.float64)[..., None]
        return np.where(ok[:, None, None], v, 0.0)

    for b in range(table.shape[0]):
        first, end = int(starts[b]), min(int(starts[b + 1]), rows)
        n, c = max(0, int(lengths[b])), min(max(0, end - first), max_count)
        for j in range(c):
            new = sorted(jj for jj in (range(j + 1) if sees is None else sees[first + j]) if jj < c)
            tokens = np.array([t for t in list(range(n)) + [n + jj for jj in new] if t < cap], np.int64)
            k, v = values(k_codes, k_scales, b, tokens), values(v_codes, v_scales, b, tokens)
            for h in range(hq):
                g = h // (hq // kvh)
                if not len(tokens):
                    out[first + j, h] = 0
                    continue
                s = k[:, g] @ q[first + j, h].astype(np.float64) / np.sqrt(dim)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[first + j, h] = p @ v[:, g]
                spread[first + j, h] = p @ np.abs(v[:, g])
                slope[first + j, h] = np.abs(k[:, g]).sum(-1).max() / np.sqrt(dim)
    return out, spread, slope
