"""NumPy restatements, in 64 bits, of the serving-step operators: chunk attention, rotary append, page fork and compaction.

Plain loops over requests, tokens and pages, written from the definitions in include/fgw_mha.h; test infrastructure only.
"""
import numpy as np


def _rows_of(table_row, positions, page):
    return [int(table_row[p // page]) * page + p % page for p in positions]


def chunk_attention(q, k_cache, v_cache, table, lens, cu, page, causal, scale):
    """(out, spread) [T, H, D] float64: the attention, and sum_j softmax_j |v_j| (what its rounding errors scale with)."""
    q, k_cache, v_cache = (np.asarray(x, dtype=np.float64) for x in (q, k_cache, v_cache))
    group = q.shape[1] // k_cache.shape[1]
    out, spread = np.zeros_like(q), np.zeros_like(q)
    for b in range(len(lens)):
        n, length = int(cu[b + 1] - cu[b]), int(lens[b])
        for i in range(n):
            seen = length - n + i + 1 if causal else length
            if seen <= 0:
                continue
            rows = _rows_of(table[b], range(seen), page)
            for h in range(q.shape[1]):
                keys, values = k_cache[rows, h // group], v_cache[rows, h // group]
                s = keys @ q[cu[b] + i, h] * scale
                if s.max() == -np.inf:  # every weight is zero: as a row that sees nothing
                    continue
                p = np.exp(s - s.max())
                p /= p.sum()
                out[cu[b] + i, h] = p @ values
                spread[cu[b] + i, h] = p @ np.abs(values)
    return out, spread


def rotary_append(q, k, v, k_cache, v_cache, table, lens, cu, cos_sin, page, interleaved):
    """(turned queries, k cache, v cache) in float64; tokens without a place give zeros and append nothing."""
    half = cos_sin.shape[1] // 2
    one = np.arange(half) * (2 if interleaved else 1)
    two = one + (1 if interleaved else half)
    q_out = np.zeros(q.shape)
    k_out, v_out = np.array(k_cache, dtype=np.float64), np.array(v_cache, dtype=np.float64)

    def turn(x, position):
        c, s = (cos_sin[position, part].astype(np.float64) for part in (slice(0, half), slice(half, None)))
        y = np.array(x, dtype=np.float64)
        y[:, one] = x[:, one] * c - x[:, two] * s
        y[:, two] = x[:, two] * c + x[:, one] * s
        return y

    for b in range(len(lens)):
        for t in range(int(cu[b]), int(cu[b + 1])):
            position = int(lens[b]) - int(cu[b + 1]) + t
            if not 0 <= position < min(table.shape[1] * page, cos_sin.shape[0]):
                continue
            q_out[t] = turn(q[t].astype(np.float64), position)
            page_id = int(table[b, position // page])
            if 0 <= page_id < k_cache.shape[0] // page:
                row = page_id * page + position % page
                k_out[row], v_out[row] = turn(k[t].astype(np.float64), position), v[t]
    return q_out, k_out, v_out


def fork_pages(table, lens, parents, reserve, page, pages):
    """(table, lens, (needed, free), copies) with copies [(src, dst, filled rows)]; the state as it was when too few
    pages are free. The first row with a parent keeps its partly filled last page if nothing else holds that page."""
    rows, width = table.shape
    kept = [int(p) if 0 <= p < rows else -1 for p in parents]
    length = [min(max(int(lens[p]), 0), width * page) if p >= 0 else 0 for p in kept]
    held = {int(e) for p, n in zip(kept, length) if p >= 0 for e in table[p, :-(-n // page)] if 0 <= e < pages}
    free = [e for e in range(pages) if e not in held]
    holds = {}  # page -> places (parent, entry) that hold it
    for p in set(kept) - {-1}:
        for w in range(-(-length[kept.index(p)] // page)):
            holds.setdefault(int(table[p, w]), []).append((p, w))
    out = np.full_like(table, -1)
    needed, copies, seen = 0, [], set()
    for i, (p, n) in enumerate(zip(kept, length)):
        if p < 0:
            continue
        room = n if reserve is None else max(min(int(reserve[i]), width * page), n)
        have = -(-n // page)
        out[i, :have] = table[p, :have]
        fresh = list(range(have, -(-room // page)))
        if n % page and (p in seen or 0 <= table[p, have - 1] < pages and len(holds[int(table[p, have - 1])]) > 1):
            fresh.insert(0, have - 1)
        for w in fresh:
            new = free[needed] if needed < len(free) else -1
            if w < have:
                copies.append((int(out[i, w]), new, n % page))
            out[i, w] = new
            needed += 1
        seen.add(p)
    if needed > len(free):
        return table.copy(), lens.copy(), (needed, len(free)), []
    copies = [c for c in copies if 0 <= c[0] < pages]
    return out, np.array(length, dtype=lens.dtype), (needed, len(free)), copies


def compact_pages(table, lens, page, pages):
    """(table, (live, moved), copies) with copies [(src, dst, rows)]."""
    rows, width = table.shape
    held = [-(-min(max(int(n), 0), width * page) // page) for n in lens]
    used = sorted({int(e) for b in range(rows) for e in table[b, :held[b]] if 0 <= e < pages})
    live = len(used)
    kept = set(used)
    holes = [e for e in range(live) if e not in kept]
    to = dict(zip([e for e in used if e >= live], holes))
    out = np.full_like(table, -1)
    for b in range(rows):
        out[b, :held[b]] = [to.get(int(e), int(e)) for e in table[b, :held[b]]]
    return out, (live, len(to)), [(src, dst, page) for src, dst in to.items()]


def copy_rows(pool, copies, page):
    """The pool after the copies (every source read as it was)."""
    out = pool.copy()
    for src, dst, rows in copies:
        out[dst * page:dst * page + rows] = pool[src * page:src * page + rows]
    return out
