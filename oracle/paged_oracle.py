"""The paged cache restated in NumPy's int64 (Python integers where products leave it), for the tests: rows are gathered, every head on its own."""
import numpy as np

from oracle import qk_oracle as o


def rows_of(pool, table_row, kv, positions):
    """[n, hd] int64 rows of one KV head at the given positions of a sequence."""
    P, at = pool.shape[2], np.asarray(positions, np.int64)
    return pool[np.asarray(table_row)[at // P], kv, at % P].astype(np.int64)


def turn(x, cos, sin, pos, rope, fa):
    """x [heads, hd] at position pos."""
    if rope == 0:
        return x
    return o.rope_fixed(x[:, None], cos[pos:pos + 1], sin[pos:pos + 1], fa, neox=rope == 2)[:, 0]


def attend(q, k, v, fa, inv_sqrt):
    """One head [hd] over rows [n, hd]."""
    if len(k) == 0:
        return np.zeros(q.shape, np.int64)
    with np.errstate(over="ignore"):
        s = (((k * q[None]).sum(1) >> fa) * np.int64(inv_sqrt)) >> fa
        return (o.softmax_fixed(s, fa)[0] @ v) >> fa


def attention(q, kpages, vpages, table, lengths, fa, window, cos, sin, rope, pages=None, inv_sqrt=None):
    B, P, Hkv, hd = len(lengths), kpages.shape[2], kpages.shape[1], kpages.shape[3]
    H = q.shape[1] // hd
    inv_sqrt = int(round((1.0 / hd ** 0.5) * (1 << fa))) if inv_sqrt is None else inv_sqrt
    out = np.zeros((B, H, hd), np.int64)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        qr = turn(q[b].reshape(H, hd), cos, sin, n - 1, rope, fa)
        lo = max(0, n - window) if window else 0
        for g in range(Hkv):
            seen = [t for t in range(lo, n)] if pages is None else [p * P + r for p in pages[b, g] if p >= 0 for r in range(P) if lo <= p * P + r < n]
            k, v = rows_of(kpages, table[b], g, seen), rows_of(vpages, table[b], g, seen)
            for h in range(g * (H // Hkv), (g + 1) * (H // Hkv)):
                out[b, h] = attend(qr[h], k, v, fa, inv_sqrt)
    return out.reshape(B, -1)


def append(k, v, kpages, vpages, bounds, table, start, rows, fa, cos, sin, rope):
    """In place."""
    P, Hkv, hd = kpages.shape[2], kpages.shape[1], kpages.shape[3]
    for b, at in enumerate(start):
        lo, hi = (b, b + 1) if rows is None else (rows[b], rows[b + 1])
        if at < 0 or hi <= lo:
            continue
        for r in range(lo, hi):
            t = at + r - lo
            kpages[table[b][t // P], :, t % P] = turn(k[r].reshape(Hkv, hd).astype(np.int64), cos, sin, t, rope, fa).astype(np.int32)
            vpages[table[b][t // P], :, t % P] = v[r].reshape(Hkv, hd).astype(np.int32)
        end = at + hi - lo
        for logical in range(at // P, (end - 1) // P + 1):
            page = table[b][logical]
            seen = kpages[page, :, :min(P, end - logical * P)]
            bounds[page, :, 0], bounds[page, :, 1] = seen.max(1), seen.min(1)


def select(q, bounds, table, lengths, P, n_select, keep_first, keep_last, fa, window, cos, sin, rope):
    B, Hkv, hd = len(lengths), bounds.shape[1], bounds.shape[3]
    H = q.shape[1] // hd
    out = np.full((B, Hkv, n_select), -1, np.int32)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        qr = turn(q[b].reshape(H, hd), cos, sin, n - 1, rope, fa)
        shown = list(range((max(0, n - window) if window else 0) // P, (n - 1) // P + 1))
        for g in range(Hkv):
            score = []
            for i, p in enumerate(shown):
                mx, mn = (bounds[table[b][p], g, s].astype(np.int64) for s in (0, 1))
                with np.errstate(over="ignore"):
                    best = max(int(np.where(qr[h] > 0, qr[h] * mx, qr[h] * mn).sum()) for h in range(g * (H // Hkv), (g + 1) * (H // Hkv)))
                score.append((1, 0) if i < keep_first or i >= len(shown) - keep_last else (0, best))
            order = sorted(range(len(shown)), key=lambda i: (-score[i][0], -score[i][1], i))[:n_select]
            out[b, g, :len(order)] = sorted(shown[i] for i in order)
    return out
