"""The paged KV cache restated with numpy in 64 bits, from the layouts' and the operators'
definitions (include/voxhip.h, vx_paged_*): what the kernels are tested against.

A cache here is float16 [layers, pages, kv_heads, ...] in the layout of its vx_buf."""
import numpy as np

NONE = 0xFFFFFFFF


def k_shape(layers, pages, page_size, kv_heads, head_dim):
    return layers, pages, kv_heads, page_size // 16, head_dim // 8, 16, 8


def v_shape(layers, pages, page_size, kv_heads, head_dim):
    return layers, pages, kv_heads, page_size // 8, head_dim, 8


def put(cache, layer, page, head, slot, row, is_v):
    """One row [head_dim] into a slot, rounded to f16."""
    with np.errstate(over="ignore"):
        row = np.asarray(row, np.float32).astype(np.float16)
    if is_v:
        cache[layer, page, head, slot // 8, :, slot % 8] = row
    else:
        cache[layer, page, head, slot // 16, :, slot % 16] = row.reshape(-1, 8)


def page_rows(cache, layer, page, head, is_v):
    """float16 rows [page_size, head_dim] of a page."""
    x = cache[layer, page, head]
    if is_v:
        return x.swapaxes(1, 2).reshape(-1, x.shape[1])
    return x.swapaxes(1, 2).reshape(x.shape[0] * 16, -1)


def rows(cache, layer, table, head, n, is_v):
    """float64 rows [n, head_dim] of positions 0..n - 1, NaN-marked `there` beside: table entries that are no page
    hold no slots."""
    ps = cache.shape[3] * (8 if is_v else 16)
    pages = cache.shape[1]
    got, there = [], []
    for k in range(-(-n // ps)):
        page = int(table[k])
        there.append(np.full(ps, page < pages))
        got.append(page_rows(cache, layer, page if page < pages else 0, head, is_v).astype(np.float64))
    return np.concatenate(got)[:n], np.concatenate(there)[:n]


def bounds_of(x):
    """[2, head_dim] of f16 rows: least and greatest, NaN where there is one."""
    return np.stack([x.min(0), x.max(0)])


def plan(lengths, counts, tables, pool, pages, page_size, max_rows, max_count):
    """dict of slots, requests, positions, granted, tables, rows, pages, taking, rows_taking."""
    width, free = tables.shape[1], min(int(pool[0]), pages)
    out = dict(slots=np.full(max_rows, NONE, np.uint32), requests=np.full(max_rows, NONE, np.uint32),
               positions=np.full(max_rows, NONE, np.uint32), granted=np.zeros(len(lengths), np.uint32), tables=tables.copy(),
               pages=0, taking=0, rows_taking=0)
    row = wanted = 0
    for i, (a, c) in enumerate(zip(lengths.tolist(), counts.tolist())):
        begin, row = row, row + c
        if not 1 <= c <= max_count or row > max_rows or a + c > width * page_size:
            continue
        have, want = -(-a // page_size), -(-(a + c) // page_size)
        first, wanted = wanted, wanted + want - have
        if want > have and wanted > free:
            continue
        for k in range(have, want):
            out["tables"][i, k] = pool[free - (first + k - have)]
        out["granted"][i] = c
        out["pages"] += want - have
        out["taking"] += 1
        out["rows_taking"] += c
        for t in range(c):
            p = a + t
            page = int(out["tables"][i, p // page_size])
            out["requests"][begin + t] = i
            out["positions"][begin + t] = p
            if page < pages:
                out["slots"][begin + t] = page * page_size + p % page_size
    out["rows"] = min(row, max_rows)
    return out


def cut(keep, lengths, tables, pool, page_size):
    """(lengths, tables, pool) afterwards."""
    lengths, tables, pool = lengths.copy(), tables.copy(), pool.copy()
    for i in range(len(lengths)):
        stay = min(int(lengths[i]), int(keep[i]))
        for k in range(-(-stay // page_size), -(-int(lengths[i]) // page_size)):
            pool[0] += 1
            pool[pool[0]] = tables[i, k]
            tables[i, k] = NONE
        lengths[i] = stay
    return lengths, tables, pool


def attention(q, k_cache, v_cache, layer, table, base, pages=None):
    """Rows [tokens, kv_heads, group, head_dim] in 64 bits of one request whose first new token is at position base: q
    the same shape; pages: for each token and KV head, indices into the table (all where None). A row that attends to
    nothing is 0."""
    tokens, kv_heads, group, hd = q.shape
    ps = v_cache.shape[3] * 8
    out = np.zeros(q.shape)
    with np.errstate(all="ignore"):
        for h in range(kv_heads):
            k, there = rows(k_cache, layer, table, h, base + tokens, False)
            v, _ = rows(v_cache, layer, table, h, base + tokens, True)
            for t in range(tokens):
                n = base + t + 1
                some = there[:n]
                if pages is not None:
                    mine = np.zeros(-(-n // ps), bool)
                    mine[[p for p in pages[t][h] if p < len(mine)]] = True
                    some = some & np.repeat(mine, ps)[:n]
                if not some.any():
                    continue
                whole = some.all()
                s = q[t, h].astype(np.float64) @ (k[:n] if whole else k[:n][some]).T / np.sqrt(hd)
                e = np.exp(s - s.max(-1, keepdims=True))
                out[t, h] = e / e.sum(-1, keepdims=True) @ (v[:n] if whole else v[:n][some])
    return out


def scores(q, bounds, layer, table, position, page_size, head):
    """float64 of every page up to the position's: q [group, head_dim]."""
    n = position // page_size + 1
    out = np.full(n, np.nan)
    q = q.astype(np.float64)
    up, down = np.where(np.isnan(q), q, np.maximum(q, 0)).sum(0), np.where(np.isnan(q), q, np.minimum(q, 0)).sum(0)
    with np.errstate(all="ignore"):
        for p in range(n):
            if table[p] < bounds.shape[1]:
                lo, hi = bounds[layer, table[p], head].astype(np.float64)
                out[p] = (up * hi + down * lo).sum()
    return out


def select(score, budget, sinks, recent):
    """u32 [budget]: the pages that stay, in rising order."""
    n = len(score)
    kind = lambda p: 0 if p < sinks or p >= n - recent else 1 if np.isnan(score[p]) else 2  # noqa: E731
    ranked = sorted(range(n), key=lambda p: (kind(p), -score[p] if kind(p) == 2 else 0.0, p))
    got = np.full(budget, NONE, np.uint32)
    chosen = sorted(ranked[:budget])
    got[:len(chosen)] = chosen
    return got
