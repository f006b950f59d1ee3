"""Plain 64-bit forms of the paged-cache operators (numpy), for the tests."""
import numpy as np

PAGE = 64


def rows_of(pool, table, g, n):
    """The first n rows of KV head g along a page-table row: [n][head_dim] float64."""
    pages = pool[table[: -(-n // PAGE)], g] if n else pool[:0, g]
    return pages.reshape(-1, pool.shape[-1])[:n].astype(np.float64)


def attention(q, k, v, table, lengths, starts, scale, prefix_pages=(), prefix_len=0):
    """(out, lse, weights, spread): out [T][H][D]; lse [T][H]; weights [B][G][slots], what each own slot receives; spread
    [T][H][D], the sum of weight * |v|, which bounds what rounded weights change."""
    T, H, D = q.shape
    B, G = len(lengths), k.shape[1]
    rep = H // G
    out, spread, lse = np.zeros((T, H, D)), np.zeros((T, H, D)), np.full((T, H), -np.inf)
    weights = np.zeros((B, G, table.shape[1] * PAGE))
    for b in range(B):
        n, nt = int(lengths[b]), int(starts[b + 1] - starts[b])
        for g in range(G):
            kk = np.concatenate([rows_of(k, np.asarray(prefix_pages, int), g, prefix_len), rows_of(k, table[b], g, n)])
            vv = np.concatenate([rows_of(v, np.asarray(prefix_pages, int), g, prefix_len), rows_of(v, table[b], g, n)])
            for i in range(nt):
                t, seen = int(starts[b]) + i, prefix_len + max(0, n - nt + i + 1)
                if not seen:
                    continue
                x = q[t, g * rep:(g + 1) * rep].astype(np.float64) @ kk[:seen].T * scale
                m = x.max(-1, keepdims=True)
                e = np.exp(x - m)
                w = e / e.sum(-1, keepdims=True)
                lse[t, g * rep:(g + 1) * rep] = (m + np.log(e.sum(-1, keepdims=True)))[:, 0]
                out[t, g * rep:(g + 1) * rep] = w @ vv[:seen]
                spread[t, g * rep:(g + 1) * rep] = w @ np.abs(vv[:seen])
                weights[b, g, : seen - prefix_len] += w[:, prefix_len:].sum(0)
    return out, lse, weights, spread


def rotate(x, gain, pos, eps, base):
    """RMS norm of every head (gain None: none) and the rotation of adjacent pairs; x [T][heads][D]."""
    x = x.astype(np.float64)
    D = x.shape[-1]
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    ang = pos.astype(np.longdouble)[:, None] * np.longdouble(base) ** (-np.arange(0, D, 2, dtype=np.longdouble) / D)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * (np.cos(ang) + 1j * np.sin(ang)).astype(np.complex128)[:, None]
    y = np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = z.real, z.imag
    return y


def evict(pos, mass, n, budget, recent):
    """(freed slots, slots of the rows that move there) of one (sequence, KV head)."""
    if n <= budget:
        return [], []
    edge = max(int(p) for p in pos[:n]) - recent
    w = [float("-inf") if m != m else float(m) for m in mass[:n]]
    kept = set(sorted(range(n), key=lambda j: (int(pos[j]) <= edge, -w[j], j))[:budget])
    return [j for j in range(budget) if j not in kept], [j for j in range(budget, n) if j in kept]
