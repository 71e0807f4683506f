"""Attention over the 4-bit KV cache where numbers span many binades: scores far below zero, keys and values
that differ by large powers of two from key to key, from half to half of a head and from row to row, and
such keys among those that a row does not see.  All against the 64-bit oracle and its bound.

The bound (oracle/kv4_oracle.py) counts fp16 terms as relative to what they stand for.  A term's low part is
also no finer than 2^-24 of its scale, half a step of it 2^-25, and the kernels take one scale for several numbers
where these differ little: that adds, in the worst case, with e = 2^-24,
  few rows, weights: steps within 2^9 of the largest of them: the largest product 2 w h of a row is at least 2^5,
      each weight is off by 2^-21 more (elements that meet 16 (c - 8) count 16-fold) and meets |c - 8| <= 8: n 2^-18,
      where sum p (h |u| + |z|) is at least 2^4 in these units: 4 n e of it;
  many rows: keys and values within 2^11 of the largest of them (each of its 15 h + |z|, at most 15 (h |u| + |z|)):
      2^-39 2^11 15 = 16 2^-28, 1 e, for a key, a value, and each of n weights;
  queries: a head's halves within 2^7: 64 x 2^-21 x 16 h / 2^(14 - 7) = 64 e of A for few rows, less for many.
"""
import numpy as np
import pytest

import test_gpu_kv4 as G
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu

F = np.float32


def _extra(q, pairs, pos, Lmax):
    """The terms above: (2 x 64 A + 4 n + 2) e of sum p (h |u| + |z|), as attention_bound lays it out."""
    (ck, cv), (zk, zv), (hk, hv) = pairs
    rep = lambda x: np.repeat(x, 64, -1)  # noqa: E731
    uk, uv = np.abs(2 * ck - 15) * rep(hk) + np.abs(rep(zk)), np.abs(2 * cv - 15) * rep(hv) + np.abs(rep(zv))
    K = rep(zk) + rep(hk) * (2 * ck - 15)
    B, M, H, hd = q.shape
    out = np.zeros(q.shape)
    for b in range(B):
        for m in range(M):
            p = int(pos[b]) + m
            if not 0 <= p < Lmax:
                continue
            for n in range(H):
                j, x = n // (H // ck.shape[1]), q[b, m, n].astype(np.float64) / np.sqrt(hd)
                A = (uk[b, j, :p + 1] @ np.abs(x)).max()
                s = K[b, j, :p + 1] @ x
                w = np.exp(s - s.max())
                out[b, m, n] = (128 * A + 4 * (p + 1) + 2) * 2.0 ** -24 * (w @ uv[b, j, :p + 1] / w.sum())
    return out


def _bounds(q, pairs, pos, Lmax):
    """The result in 64 bits, and how far from it an element may be."""
    K, V = ((z.repeat(64, -1) + h.repeat(64, -1) * (2 * c - 15)) for c, z, h in zip(*pairs))
    return K4.attention(q, K, V, pos, Lmax), K4.attention_bound(q, *pairs, pos, Lmax) + _extra(q, pairs, pos, Lmax) + 1e-37


def _check(hip, q, cache, pairs, pos, Lmax, y=None):
    """Every element within the bound; the whole, row by row, within a quarter of it (roundings are as often up as
    down)."""
    import torch

    if y is None:
        out = hip.kv4_attention(*G._cuda(q), cache, G._pos(pos), max_len=Lmax)
        assert torch.isfinite(out).all()
        assert torch.equal(out, hip.kv4_attention(*G._cuda(q), cache, G._pos(pos), max_len=Lmax))
        y = out.cpu().numpy()
    want, bound = _bounds(q, pairs, pos, Lmax)
    off = np.abs(y - want)
    assert np.isfinite(y).all()
    assert (off <= bound).all(), f"off by {np.max(off / bound):.3g} bounds"
    rows = lambda x: np.linalg.norm(x.reshape(-1, 64), axis=-1)  # noqa: E731
    assert (rows(off) <= 0.25 * rows(bound)).all(), f"a row is off by {np.max(rows(off) / rows(bound)):.3g} bounds"
    return y, want


# (B, M, H, Hkv, hd, Lmax, positions of row 0, written positions)
FEW = [
    # tiles of 4 rows: one block, part of one, splits; queries of one head
    (1, 1, 20, 5, 128, 640, [0], 1),
    (1, 1, 20, 5, 128, 640, [70], 71),
    (1, 1, 20, 5, 128, 2048, [1537], 1538),
    (1, 4, 2, 2, 64, 300, [62], 66),
    # of 8, across a block's border, and in splits
    (1, 2, 20, 5, 128, 640, [63], 65),
    (1, 4, 8, 4, 64, 2000, [700], 704),
    # of 16, with four waves and with eight
    (1, 4, 20, 5, 128, 640, [62], 66),
    (2, 30, 14, 2, 64, 200, [0, 100], 130),
    (1, 16, 20, 5, 128, 900, [60], 76),
    (2, 30, 14, 2, 64, 1500, [0, 800], 830),
    # splits by length
    (5, 1, 20, 5, 128, 3000, [1500, 0, 1200, 64, -1], 1501),
    (3, 4, 8, 2, 64, 2000, [1996, 1, 1990], 2000),
]
MANY = [
    (1, 64, 20, 5, 128, 20000, [64], 128),
    (1, 100, 20, 5, 128, 20000, [0], 100),
    (2, 73, 14, 2, 64, 98000, [0, 301], 374),
    (1, 200, 3, 3, 128, 57000, [70], 270),
    (2, 90, 4, 2, 128, 57000, [-50, 40], 130),
]


def _far(seed, B, M, n, H, Hkv, hd, nats):
    """Queries and keys whose scores all lie about `nats` below zero, and values."""
    q, _, _ = G._inputs(seed, B, M, H, Hkv, hd)
    _, k, v = G._inputs(seed + 1, B, n, H, Hkv, hd)
    side = F(np.sqrt(nats / np.sqrt(hd)))  # q . k = -side^2 hd = -nats sqrt(hd)
    return q * F(0.3) + side, k * F(0.3) - side, v


@pytest.mark.parametrize("nats", [100, 300])
@pytest.mark.parametrize("case", FEW + MANY)
def test_scores_far_below_zero(hip, case, nats):
    """A softmax does not hang on a common offset of its scores."""
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, k, v = _far(B * 100 + M, B, M, n, H, Hkv, hd, nats)
    cache, pairs = G._filled(hip, 0, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    _check(hip, q, cache, pairs, pos, Lmax)


def _step(hip, q, k, v, cache, pos, Lmax):
    """kv4_step of the rows at pos (angles 0), over a cache that holds them already."""
    import torch

    B, hd = q.shape[0], q.shape[-1]
    table = np.zeros((Lmax, hd // 2, 2), F)
    table[..., 0] = 1
    at = np.clip(pos, 0, k.shape[1] - 1)
    new = [np.stack([x[b, at[b]] for b in range(B)])[:, None] for x in (k, v)]
    copy = cache.clone()
    y = hip.kv4_step(*G._cuda(q, *new), copy, *G._cuda(table), G._pos(pos), max_len=Lmax)
    assert torch.equal(copy, cache)
    return y.cpu().numpy()


@pytest.mark.parametrize("nats", [100, 300])
@pytest.mark.parametrize("case", [c for c in FEW if c[1] == 1])
def test_step_scores_far_below_zero(hip, case, nats):
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, k, v = _far(B * 100 + M, B, M, n, H, Hkv, hd, nats)
    cache, pairs = G._filled(hip, 0, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    _check(hip, q, cache, pairs, pos, Lmax, y=_step(hip, q, k, v, cache, pos, Lmax))


def _parts(case):
    """Queries, keys and values of a case and, for each sequence, a key in its middle: the last rows see it, the
    first do not (one token: it does)."""
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, _, _ = G._inputs(B * 7 + M, B, M, H, Hkv, hd)
    _, k, v = G._inputs(B * 100 + M, B, n, H, Hkv, hd)
    at = [p + M // 2 if M > 1 else p // 2 for p in pos]
    return q, k, v, [(b, p) for b, p in enumerate(at) if 0 <= p < n]


def _attend(hip, case, q, k, v):
    B, M, H, Hkv, hd, Lmax, pos, n = case
    with np.errstate(over="ignore"):
        cache, pairs = G._filled(hip, 0, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    y, _ = _check(hip, q, cache, pairs, pos, Lmax)
    if M == 1:
        assert np.array_equal(_step(hip, q, k, v, cache, pos, Lmax), y)
    return y, cache


@pytest.mark.parametrize("case", FEW + MANY)
def test_blocks_of_values_far_apart(hip, case):
    """Every other block of 64 positions holds values of 2^90, the rest of 2^-60: their waves and splits meet in
    the join."""
    q, k, v, _ = _parts(case)
    even = (np.arange(v.shape[1]) // 64 % 2 == 0)[None, :, None, None]
    _attend(hip, case, q, k, np.where(even, np.ldexp(v, 90), np.ldexp(v, -60)))


@pytest.mark.parametrize("d", [20, 22, 23, 24, 25, 26, 30, 60])
@pytest.mark.parametrize("case", FEW + MANY)
def test_large_scores(hip, case, d):
    """Scores of some 2^d: one key has all the weight."""
    q, k, v, _ = _parts(case)
    _attend(hip, case, q, np.ldexp(k, d - 1), v)


@pytest.mark.parametrize("d", [20, 40, 80])
@pytest.mark.parametrize("which", ["v", "k", "both"])
@pytest.mark.parametrize("case", FEW + MANY)
def test_outlier(hip, case, which, d):
    """A key 2^d as large as the others that half of the rows see: it is nothing to the other half."""
    q, k, v, at = _parts(case)
    for b, p in at:
        if which != "k":
            v[b, p] = np.ldexp(v[b, p], d)
        if which != "v":
            k[b, p] = np.ldexp(k[b, p], d)
    _attend(hip, case, q, k, v)


def _little(case, nats, d):
    """The keys in the middle `nats` above (below zero: below) the others' scores, their values times 2^d."""
    q, k, v, at = _parts(case)
    q = q * F(0.3) + 1
    for b, p in at:
        k[b, p] = nats / np.sqrt(q.shape[-1])
        v[b, p] = np.ldexp(v[b, p], d)
    return q, k, v


@pytest.mark.parametrize("d", [20, 40, 55])
@pytest.mark.parametrize("case", FEW + MANY)
def test_outlier_of_little_weight(hip, case, d):
    """Values 2^d as large as the others under weights of 2^-60."""
    _attend(hip, case, *_little(case, -42, d))


@pytest.mark.parametrize("d", [-200, -40, -12])
@pytest.mark.parametrize("case", FEW + MANY)
def test_weight_on_a_key_of_little_value(hip, case, d):
    """One key has nearly all the weight and next to no value (or none): the rest of 2^-60 is the result."""
    _attend(hip, case, *_little(case, 42, d))


@pytest.mark.parametrize("d", [8, 30, 60])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("which", ["v", "k", "q", "qk"])
@pytest.mark.parametrize("case", [c for c in FEW + MANY if c[4] == 128])
def test_halves_of_a_head_far_apart(hip, case, which, side, d):
    """One group of 64 dimensions is 2^d as large as the other (queries: 2^-d)."""
    q, k, v, _ = _parts(case)
    part = np.s_[..., 64 * side:64 * side + 64]
    if "q" in which:
        q[part] = np.ldexp(q[part], -d)
    if "k" in which:
        k[part] = np.ldexp(k[part], d)
    if "v" in which:
        v[part] = np.ldexp(v[part], d)
    _attend(hip, case, q, k, v)


@pytest.mark.parametrize("d", [-115, 90])
@pytest.mark.parametrize("case", FEW + MANY)
def test_values_of_any_size(hip, case, d):
    q, k, v, _ = _parts(case)
    _attend(hip, case, q, k, np.ldexp(v, d))


@pytest.mark.parametrize("kd", [-2000, -60, -20])
@pytest.mark.parametrize("case", FEW + MANY)
def test_zero_queries(hip, case, kd):
    """Queries of 0, over keys of 0 or small ones: the mean of the values."""
    q, k, v, _ = _parts(case)
    _attend(hip, case, 0 * q, np.ldexp(k, kd), v)


@pytest.mark.parametrize("case", [c for c in FEW + MANY if c[1] > 1])
def test_nan_next_to_an_outlier(hip, case):
    """A NaN that a row does not see leaves every bit of it also where the block holds an outlier."""
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, k, v, at = _parts(case)
    for b, p in at:
        v[b, p] = np.ldexp(v[b, p], 40)
    y, cache = _attend(hip, case, q, k, v)
    pairs = [K4.quantise(x.transpose(0, 2, 1, 3)) for x in (k, v)]
    want, bound = _bounds(q, list(zip(*pairs)), pos, Lmax)
    seen = np.zeros(y.shape, bool)
    for b, p in at:
        k[b, p, 0, 3], v[b, p, -1, 1] = np.nan, np.inf
        rows = pos[b] + np.arange(M)
        rows = (rows >= p) & (rows < Lmax)
        seen[b, rows, :H // Hkv] = True
        seen[b, rows, H - H // Hkv:, :64] = True
    cache, _ = G._filled(hip, 0, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    z = hip.kv4_attention(*G._cuda(q), cache, G._pos(pos), max_len=Lmax).cpu().numpy()
    assert np.isnan(z[seen]).all()
    if hd == 64:  # (the last head's NaN takes the outlier's place, and with it the reason for other terms)
        last = np.s_[:, :, H - H // Hkv:]
        far = np.abs(z[last] - want[last]) <= bound[last]
        assert (far | seen[last]).all()
        z[last] = y[last]
    assert np.array_equal(z[~seen], y[~seen])


@pytest.mark.parametrize("case", [c for c in FEW + MANY if c[1] > 1])
def test_in_place_with_an_outlier(hip, case):
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, k, v, at = _parts(case)
    for b, p in at:
        v[b, p] = np.ldexp(v[b, p], 40)
    y, cache = _attend(hip, case, q, k, v)
    (t,) = G._cuda(q)
    assert hip.kv4_attention(t, cache, G._pos(pos), max_len=Lmax, out=t) is t
    assert np.array_equal(t.cpu().numpy(), y)


@pytest.mark.parametrize("x", [np.nan, np.inf])
@pytest.mark.parametrize("case", [c for c in FEW + MANY if c[4] == 128 and c[2] > c[3]])
def test_query_that_is_no_number(hip, case, x):
    """Its row is NaN, every other row keeps every bit."""
    B, M, H, Hkv, hd, Lmax, pos, n = case
    q, k, v, _ = _parts(case)
    y, cache = _attend(hip, case, q, k, v)
    q[0, M - 1, 1, 77] = x
    y[0, M - 1, 1] = np.nan
    z = hip.kv4_attention(*G._cuda(q), cache, G._pos(pos), max_len=Lmax).cpu().numpy()
    assert np.array_equal(z, y, equal_nan=True)


@pytest.mark.parametrize("which", ["v", "k", "q"])
def test_tiles_of_256_rows_without_splits(hip, which):
    """A batch that fills the GPU: no join, results straight from the tiles, in place too; three sequences of 129
    against the oracle."""
    B, M, H, Hkv, hd, Lmax, n = 129, 64, 8, 2, 128, 600, 100
    assert hip.lib.rt_kv4_attention_workspace(B, M, H, Hkv, hd, Lmax) == 0
    pos = [(b * 7) % 37 for b in range(B)]
    case = (B, M, H, Hkv, hd, Lmax, pos, n)
    q, k, v, at = _parts(case)
    for b, p in at[::2]:
        if which == "v":
            v[b, p] = np.ldexp(v[b, p], 40)
        elif which == "k":
            k[b, p] = np.ldexp(k[b, p], 40)
        else:
            q[b, 5, :, 64:] = np.ldexp(q[b, 5, :, 64:], -30)
            k[b, :, :, 64:] = np.ldexp(k[b, :, :, 64:], 30)
    cache, pairs = G._filled(hip, 0, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    (t,) = G._cuda(q)
    y = hip.kv4_attention(t, cache, G._pos(pos), max_len=Lmax)
    assert hip.kv4_attention(t, cache, G._pos(pos), max_len=Lmax, out=t) is t
    assert np.array_equal(t.cpu().numpy(), y.cpu().numpy())
    for b in (0, 64, 65, 128):
        sub = [tuple(x[b:b + 1] for x in p) for p in pairs]
        _check(hip, q[b:b + 1], None, sub, pos[b:b + 1], Lmax, y=y[b:b + 1].cpu().numpy())
