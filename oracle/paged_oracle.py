"""The paged KV cache by its definition, in 64 bits, slot by slot (test infrastructure).

cache: [2 (K, V), pages, Hkv, page, hd] (a CPU tensor of the cache's type); slot t of sequence b is row t % page of page
table[b][t // page], and is there if t < lens[b] and that number is a page's.
"""
import torch


def page_of(cache, table, b, t):
    """The page of slot t of sequence b, or None."""
    page = cache.shape[3]
    if not 0 <= t < table.shape[1] * page:
        return None
    n = int(table[b, t // page])
    return n if 0 <= n < cache.shape[1] else None


def rotate(x, angles, interleaved):
    """x float64 [.., hd] by angles [rotary / 2, 2] = (cos, sin)."""
    n = angles.shape[0]
    at = [(2 * i, 2 * i + 1) if interleaved else (i, i + n) for i in range(n)]
    a, b = [p[0] for p in at], [p[1] for p in at]
    c, s = angles.double().unbind(-1)
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def append(q, k, v, cache, table, lens, rope, pos, counts=None, interleaved=False):
    """(rotated q, {(page, row): (key, value)} float64 [Hkv, hd] of what is written): the cache is not changed."""
    out, rows = torch.zeros(q.shape, dtype=torch.float64), {}
    page = cache.shape[3]
    for b in range(q.shape[0]):
        for m in range(q.shape[1] if counts is None else min(q.shape[1], int(counts[b]))):
            p, t = int(pos[b]) + m, int(lens[b]) + m
            n = page_of(cache, table, b, t)
            if n is None or not 0 <= p < rope.shape[0]:
                continue
            out[b, m] = rotate(q[b, m].double(), rope[p], interleaved)
            rows[n, t % page] = rotate(k[b, m].double(), rope[p], interleaved), v[b, m].double()
    return out, rows


def attend(q, cache, table, lens):
    """(o float64 [B, 1, H, hd], weights [B, Hkv, P * page] summed over each KV head's query heads, and per output what its
    error is counted against: sum p |v| and the largest sum |q k| / sqrt(hd) of its scores)."""
    B, _, H, hd = q.shape
    Hkv, page = cache.shape[2:4]
    G, cap = H // Hkv, table.shape[1] * page
    o, weights, size, most = (torch.zeros(s, dtype=torch.float64) for s in (q.shape, (B, Hkv, cap), q.shape, (B, 1, H, 1)))
    for b in range(B):
        there = [(t, n) for t in range(min(int(lens[b]), cap)) if (n := page_of(cache, table, b, t)) is not None]
        if not there:
            continue
        t, n = (torch.tensor(x) for x in zip(*there))
        K, V = (x.double() for x in cache[:, n, :, t % page].unbind(1))  # [L, Hkv, hd]
        for h in range(H):
            x, kv = q[b, 0, h].double(), h // G
            p = torch.softmax(K[:, kv] @ x / hd ** 0.5, 0)
            o[b, 0, h], size[b, 0, h] = p @ V[:, kv], p @ V[:, kv].abs()
            most[b, 0, h] = (K[:, kv].abs() @ x.abs()).max() / hd ** 0.5
            weights[b, kv, t] += p
    return o, weights, size, most


def evict(cache, table, lens, weights, keep, recent):
    """For every sequence and KV head the slots that are kept, in order."""
    B, Hkv, _ = weights.shape
    kept = []
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * cache.shape[3])
        there = [t for t in range(n) if page_of(cache, table, b, t) is not None]
        stay = [t for t in there if t >= n - recent]
        judged = [t for t in there if t < n - recent]

        def order(w):  # NaN counts as the largest
            return float("inf") if w != w else w

        kept.append([])
        for h in range(Hkv):
            w = [float(x) for x in weights[b, h]]
            best = sorted(judged, key=lambda t: (w[t] == w[t], -order(w[t]), t))[:keep - len(stay)]
            kept[-1].append(sorted(best) + stay)
    return kept
