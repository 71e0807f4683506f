"""The 4-bit KV cache on the GPU: what is written and read back equals its definition bit for bit,
and attention over it is within derived bounds of the same formula in 64 bits (oracle/kv4_oracle.py)."""
import numpy as np
import pytest

from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu

THETA = 500000.0


def _rope(Lmax, hd):
    from rotor.bitnet_model import rope_table

    return rope_table(Lmax, hd, THETA)


def _inputs(seed, B, M, H, Hkv, hd):
    """Queries, keys and values; one channel in sixteen is four times as wide and keys have a mean."""
    rng = np.random.default_rng(seed)
    wide = np.where(rng.random((1, 1, Hkv, hd)) < 1 / 16, 4, 1)
    q = rng.standard_normal((B, M, H, hd)).astype(np.float32)
    k = (rng.standard_normal((B, M, Hkv, hd)) * wide + 0.5 * rng.standard_normal((Hkv, hd))).astype(np.float32)
    v = rng.standard_normal((B, M, Hkv, hd)).astype(np.float32)
    return q, k, v


def _cuda(*xs):
    import torch

    return [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in xs]


def _pos(pos):
    import torch

    return torch.tensor(pos, dtype=torch.int32, device="cuda")


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def _zeros_pos(B):
    return _pos([0] * B)


# (B, M, H, Hkv, hd, Lmax, positions): one token, runs that end inside blocks of 16 and 64, rows in front of
# the cache and behind it, one query head a KV head and many
WRITES = [
    (1, 1, 20, 5, 128, 640, [0]),
    (1, 1, 20, 5, 128, 640, [639]),
    (1, 1, 2, 1, 64, 64, [17]),
    (3, 2, 6, 2, 64, 100, [15, 63, 98]),
    (2, 15, 4, 4, 128, 130, [0, 115]),
    (2, 16, 4, 2, 128, 130, [16, 9]),
    (2, 17, 7, 1, 64, 200, [31, 64]),
    (1, 63, 8, 2, 128, 300, [1]),
    (2, 64, 3, 3, 64, 300, [64, 5]),
    (1, 130, 20, 5, 128, 1000, [777]),
    (5, 3, 4, 2, 64, 70, [-1, -3, 69, 70, 68]),
    (4, 40, 4, 2, 128, 90, [-20, 80, -40, 1000]),
    (3, 2, 4, 2, 64, 64, [2147483647, -2147483648, 62]),
]


@pytest.mark.parametrize("B,M,H,Hkv,hd,Lmax,pos", WRITES)
def test_append_and_read(hip, B, M, H, Hkv, hd, Lmax, pos):
    import torch

    q, k, v = _inputs(B * 1000 + M, B, M, H, Hkv, hd)
    table = _rope(Lmax, hd)
    cache = hip.kv4_cache(Hkv, hd, Lmax, batch=B)
    cache.random_(0, 256)
    # scales of what is not written: finite numbers, so that they compare
    cache.view(torch.int32)[..., 16 * hd:] &= 0x3FFF3FFF
    before = [x.cpu().numpy() for x in hip.kv4_read(cache, _zeros_pos(B), Lmax, max_len=Lmax)]
    tq, tk, tv, trope = _cuda(q, k, v, table)
    y = hip.kv4_append(tq, tk, tv, cache, trope, _pos(pos), max_len=Lmax).cpu().numpy()
    after = [x.cpu().numpy() for x in hip.kv4_read(cache, _zeros_pos(B), Lmax, max_len=Lmax)]
    rows = [x.cpu().numpy() for x in hip.kv4_read(cache, _pos(pos), M, max_len=Lmax)]
    assert torch.equal(tq.cpu(), torch.from_numpy(q)) and torch.equal(tk.cpu(), torch.from_numpy(k))
    want, want_q = [x.copy() for x in before], np.zeros_like(q)
    want_rows = [np.zeros((B, Hkv, M, hd), np.float32) for _ in range(2)]
    for b in range(B):
        for m in range(M):
            p = pos[b] + m
            if not 0 <= p < Lmax:
                continue
            want_q[b, m] = K4.rope(q[b, m], table, p)
            for i, x in enumerate((K4.rope(k[b, m], table, p), v[b, m])):
                want[i][b, :, p] = want_rows[i][b, :, m] = K4.held(x)
    assert _same(y, want_q)
    for i in range(2):
        assert _same(after[i], want[i])
        assert _same(rows[i], want_rows[i])


@pytest.mark.parametrize("hd", [64, 128])
def test_append_special_groups(hip, hd):
    """Zeros, constants, NaN, infinities, the largest and the smallest numbers, ties between levels."""
    rng = np.random.default_rng(hd)
    M, Lmax = 40, 64
    v = rng.standard_normal((1, M, 1, hd)).astype(np.float32)
    v[0, 0], v[0, 1], v[0, 2, 0, 3], v[0, 3, 0, 5], v[0, 4] = 0, 2.5, np.nan, -np.inf, 3.4e38
    v[0, 5, 0, ::2], v[0, 5, 0, 1::2] = 3e38, -3e38
    v[0, 6] *= 1e-38
    v[0, 7] *= 1e-44
    v[0, 8] = -0.0
    v[0, 9] += 1e6
    v[0, 10, 0, :64] = np.arange(64) % 29 - 14
    v[0, 10, 0, :2] = -15, 15
    for j in range(11, 40):  # numbers on and next to the borders between levels of the group's own z and h
        c, z, h = K4.quantise(v[0, j, 0, :64])
        border = (z[0] + h[0] * (2 * rng.integers(0, 15, 40) - 14)).astype(np.float32)
        side = rng.integers(-1, 2, 40)
        v[0, j, 0, 12:52] = np.where(side == 0, border, np.nextafter(border, np.float32(3e38) * side.astype(np.float32)))
    k = v[:, ::-1].copy()
    table = _rope(Lmax, hd)
    table[..., 0], table[..., 1] = 1, 0  # keys as they are
    q = rng.standard_normal((1, M, 1, hd)).astype(np.float32)
    cache = hip.kv4_cache(1, hd, Lmax)
    hip.kv4_append(*_cuda(q, k, v), cache, *_cuda(table), _pos([9]))
    got = [x.cpu().numpy()[0, 0] for x in hip.kv4_read(cache, _pos([9]), M)]
    with np.errstate(all="ignore"):
        assert _same(got[0], K4.held(K4.rope(k[0], table, 0)[:, 0]))
    assert _same(got[1], K4.held(v[0, :, 0]))


def test_token_by_token_equals_at_once(hip):
    """The cache's bytes do not hang on how the tokens came in, and neither do rows computed twice."""
    import torch

    B, M, H, Hkv, hd, Lmax = 2, 150, 4, 2, 128, 200
    q, k, v = _cuda(*_inputs(3, B, M, H, Hkv, hd))
    (rope,) = _cuda(_rope(Lmax, hd))
    base = torch.randint(0, 256, (B, Hkv, 4, 72 * hd), dtype=torch.uint8, device="cuda")
    one, many, odd = base.clone(), base.clone(), base.clone()
    start = torch.tensor([3, 49], dtype=torch.int32, device="cuda")
    y = hip.kv4_append(q, k, v, one, rope, start)
    for m in range(M):
        z = hip.kv4_append(q[:, m:m + 1], k[:, m:m + 1], v[:, m:m + 1], many, rope, start + m)
        assert torch.equal(z[:, 0], y[:, m])
    for m in range(0, M, 37):
        hip.kv4_append(q[:, m:m + 37], k[:, m:m + 37], v[:, m:m + 37], odd, rope, start + m)
    assert torch.equal(one, many) and torch.equal(one, odd)
    hip.kv4_append(q, k, v, one, rope, start)
    assert torch.equal(one, many)


def test_layout(hip):
    """Where codes and scales lie, read from the bytes by the description in the kernels' source."""
    B, L, Hkv = 1, 128, 2
    for hd in (64, 128):
        q, k, v = _inputs(hd, B, L, Hkv, Hkv, hd)
        table = _rope(L, hd)
        cache = hip.kv4_cache(Hkv, hd, L)
        hip.kv4_append(*_cuda(q, k, v), cache, *_cuda(table), _pos([0]))
        words = cache.cpu().numpy().view(np.uint32)
        rk = np.stack([K4.rope(k[0, p], table, p) for p in range(L)])
        for x, at, is_v in ((rk, 0, False), (v[0], 8 * hd, True)):
            c, z, h = K4.quantise(x)
            for p, n, d in [(0, 0, 0), (1, 1, 5), (77, 0, hd - 1), (63, 1, 33), (100, 1, 17), (42, 0, 40), (127, 1, hd - 9)]:
                P = p % 64
                if is_v:
                    i, e = ((d // 32 * 16 + d % 16) * 4 + P % 32 // 16 * 2 + P % 8 // 4) * 4 + d % 32 // 16 * 2 + P // 32, P % 16 // 8 * 4 + P % 4
                else:
                    i, e = P * (hd // 8) + d % 64 // 16 * (hd // 32) + d // 64 * 2 + d % 16 // 8, d % 8
                block = words[0, n, p // 64]
                assert (int(block[at + i]) >> (e // 2 * 4 + e % 2 * 16)) & 15 == c[p, n, d]
                s = int(block[16 * hd + (hd if is_v else 0) + d // 64 * 64 + P])
                f = lambda b: np.uint32(b << 16).view(np.float32)  # noqa: E731
                assert f(s >> 16) == z[p, n, d // 64] and f(s & 0xFFFF) == h[p, n, d // 64]


def _filled(hip, seed, B, H, Hkv, hd, Lmax, n, k=None, v=None):
    """A cache with positions [0, n) of every sequence written (keys as they are: no rotation), NaN codes and
    scales behind them, and its (codes, z, h) pairs from the definition."""
    _, k0, v0 = _inputs(seed, B, n, H, Hkv, hd)
    k, v = (k0 if k is None else k), (v0 if v is None else v)
    table = _rope(Lmax, hd)
    table[..., 0], table[..., 1] = 1, 0
    cache = hip.kv4_cache(Hkv, hd, Lmax, batch=B)
    cache.fill_(0xFF)
    hip.kv4_append(*_cuda(np.zeros((B, n, H, hd), np.float32), k, v), cache, *_cuda(table), _zeros_pos(B), max_len=Lmax)
    pairs = list(zip(*(K4.quantise(x.transpose(0, 2, 1, 3)) for x in (k, v))))
    return cache, pairs


def _check(hip, q, cache, pairs, pos, Lmax):
    import torch

    out = hip.kv4_attention(*_cuda(q), cache, _pos(pos), max_len=Lmax)
    again = hip.kv4_attention(*_cuda(q), cache, _pos(pos), max_len=Lmax)
    assert torch.equal(out, again)  # no result hangs on an order that changes
    y = out.cpu().numpy()
    K, V = ((z.repeat(64, -1) + h.repeat(64, -1) * (2 * c - 15)) for c, z, h in zip(*pairs))
    with np.errstate(all="ignore"):
        want = K4.attention(q, K, V, pos, Lmax)
        bound = K4.attention_bound(q, *pairs, pos, Lmax)
    off = np.abs(y - want)
    assert (off <= bound + 1e-37).all(), f"off by {np.max(off / (bound + 1e-37)):.3g} bounds"
    # roundings are as often up as down: the whole is far nearer than the sum of the worst cases
    norm = np.linalg.norm(want)
    assert norm == 0 or np.linalg.norm(off) <= 0.25 * np.linalg.norm(bound)
    return y, want


# (B, M, H, Hkv, hd, Lmax, positions of row 0, written positions)
ATTENDS = [
    (1, 1, 20, 5, 128, 640, [0], 1),
    (1, 1, 20, 5, 128, 640, [63], 64),
    (1, 1, 20, 5, 128, 640, [64], 65),
    (1, 1, 20, 5, 128, 2048, [1537], 1538),
    (1, 1, 1, 1, 64, 65, [64], 65),
    (4, 1, 12, 12, 64, 777, [776, 5, 128, 400], 777),
    (3, 1, 16, 1, 128, 300, [299, 0, 150], 300),
    (2, 1, 20, 1, 64, 300, [299, 17], 300),       # more rows than a tile of 16
    (2, 3, 14, 2, 64, 200, [100, 197], 200),
    (2, 4, 20, 5, 128, 260, [256, 0], 260),
    (1, 5, 6, 2, 128, 128, [123], 128),
    (1, 33, 4, 4, 64, 100, [0], 33),
    (1, 64, 20, 5, 128, 128, [64], 128),
    (1, 100, 20, 5, 128, 320, [0], 100),
    (2, 77, 14, 2, 64, 400, [0, 301], 378),
    (1, 130, 3, 3, 128, 200, [70], 200),
    (1, 129, 7, 1, 64, 140, [3], 132),
    (3, 2, 4, 2, 64, 64, [-1, 63, 2147483647], 64),  # rows outside the cache
    (2, 90, 4, 2, 128, 100, [-50, 40], 100),
    (2, 40, 8, 2, 64, 100, [-100, 200], 100),         # nothing but such rows
    # batches whose splits go by length: sequences of none to many blocks, 64 of them, 16 rows a tile
    (5, 1, 20, 5, 128, 3000, [2999, 0, 1200, 64, -1], 3000),
    (3, 4, 8, 2, 64, 2000, [1996, 1, 1990], 2000),
    (64, 1, 4, 2, 64, 2048, [(i * 997) % 2048 for i in range(64)], 2048),
    (2, 2, 3, 3, 128, 1500, [-2, 5000], 1500),
    (7, 1, 2, 1, 128, 1400, [1399] * 6 + [3], 1400),
]


# The same rows over long caches (a call is taken to stand at the end of its cache, and takes tiles of 256
# rows where their keys are many)
ATTENDS += [
    (1, 33, 4, 4, 64, 21000, [0], 33),
    (1, 64, 20, 5, 128, 16700, [64], 128),
    (1, 100, 20, 5, 128, 16700, [0], 100),
    (2, 77, 14, 2, 64, 10600, [0, 301], 378),
    (1, 130, 3, 3, 128, 28000, [70], 200),
    (1, 300, 2, 2, 64, 21000, [211], 511),
    (1, 129, 7, 1, 64, 21000, [3], 132),
    (2, 90, 4, 2, 128, 21000, [-50, 40], 130),   # rows in front of the cache
    (2, 40, 8, 2, 64, 21000, [-100, 30000], 1),  # nothing but rows outside it
    (1, 70, 2, 1, 64, 83250, [83210], 83250),    # rows behind it
    (3, 9, 1, 1, 128, 28000, [5, 0, 64], 73),    # nine rows
    # (... and rows enough for such tiles to pay)
    (1, 64, 20, 5, 128, 20000, [64], 128),
    (1, 100, 20, 5, 128, 20000, [0], 100),
    (2, 73, 14, 2, 64, 98000, [0, 301], 374),
    (1, 200, 3, 3, 128, 57000, [70], 270),
    (1, 250, 6, 6, 64, 130000, [261], 511),
    (1, 127, 16, 2, 64, 98000, [3], 130),
    (2, 90, 4, 2, 128, 57000, [-50, 40], 130),
    (2, 64, 32, 8, 64, 50000, [-100, 70000], 1),
    (1, 64, 12, 3, 128, 33000, [32960], 33000),
    # eight waves a workgroup: blocks for some, all or none of them
    (1, 16, 20, 5, 128, 900, [884], 900),
    (2, 30, 14, 2, 64, 1000, [0, 700], 730),
    (1, 3, 16, 2, 128, 833, [447], 450),
    (1, 64, 20, 5, 128, 2600, [2500], 2564),  # ... in splits
    (2, 30, 14, 2, 64, 1500, [0, 1300], 1330),
    # many sequences of few rows: tiles of 16
    (40, 5, 8, 2, 64, 700, [(i * 97) % 690 for i in range(40)], 700),
    (130, 3, 20, 5, 128, 300, [(i * 31) % 298 for i in range(130)], 300),
]


@pytest.mark.parametrize("B,M,H,Hkv,hd,Lmax,pos,n", ATTENDS)
def test_attention(hip, B, M, H, Hkv, hd, Lmax, pos, n):
    cache, pairs = _filled(hip, B * 100 + M, B, H, Hkv, hd, Lmax, n)
    q, _, _ = _inputs(B * 7 + M, B, M, H, Hkv, hd)
    y, _ = _check(hip, q, cache, pairs, pos, Lmax)
    for b in range(B):
        for m in range(M):
            assert 0 <= pos[b] + m < Lmax or (y[b, m] == 0).all()


@pytest.mark.parametrize("M,Lmax", [(1, 300), (1, 4000), (3, 300), (70, 300), (70, 21000), (64, 50000)])
@pytest.mark.parametrize("qs,ks,vs", [(1e-30, 1, 1), (20, 1, 1), (1, 1e-20, 1), (1e-15, 1e15, 1), (1, 1, 1e-25), (1, 1, 1e25),
                                      (0, 1, 1), (1, 0, 0)])
def test_attention_scales(hip, M, Lmax, qs, ks, vs):
    """Queries, keys and values of any size, zero among them."""
    B, H, Hkv, hd, n = 1, 8, 2, 128, 290
    q, k, v = _inputs(M, B, n, H, Hkv, hd)
    f = np.float32
    cache, pairs = _filled(hip, 5, B, H, Hkv, hd, Lmax, n, k=k * f(ks), v=v * f(vs))
    _check(hip, q[:, :M] * f(qs), cache, pairs, [n - M], Lmax)


@pytest.mark.parametrize("M,Lmax", [(1, 700), (1, 2000), (40, 700), (40, 83300), (64, 800000)])
def test_attention_values_of_very_different_sizes(hip, M, Lmax):
    """The weights' fp16 terms are scaled by the largest step of the values seen: outliers, early and late, that
    weigh little do not take the others' bits."""
    B, H, Hkv, hd, n = 1, 4, 1, 64, 700
    q, k, v = _inputs(11, B, n, H, Hkv, hd)
    v *= np.exp2(np.random.default_rng(2).integers(-8, 9, (B, n, 1, 1))).astype(np.float32)
    v[:, [3, 400, 650]] *= 1000
    cache, pairs = _filled(hip, 5, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    _check(hip, q[:, :M], cache, pairs, [n - M], Lmax)


@pytest.mark.parametrize("M,Lmax", [(1, 8192), (24, 8192), (24, 42000), (64, 50000)])
def test_attention_long_and_even(hip, M, Lmax):
    """8192 keys that weigh about the same: the result is a small difference of large sums.  In 64 bits against
    fp32 sums of numbers with random signs: each of 2 x 8192 terms (magnitude at most 3 of the values' deviation)
    is off by 2^-24 of a running sum no larger than that of the result's own order times 8192; the relative error's
    deviation is below 2^-24 x sqrt(2 x 8192) = 8e-6 even if every rounding were a full half step of the largest
    running sum, and rounding errors of that size are rarer: 2e-6 is asked for (the plain fp32 form has 1e-6)."""
    B, H, Hkv, hd, n = 1, 8, 2, 128, 8192
    q, k, v = _inputs(4, B, n, H, Hkv, hd)
    cache, pairs = _filled(hip, 5, B, H, Hkv, hd, Lmax, n, k=np.float32(0.05) * k, v=v)
    y, want = _check(hip, q[:, :M], cache, pairs, [n - M], Lmax)
    assert np.linalg.norm(y - want) <= 2e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("M,Lmax", [(1, 200), (1, 3000), (9, 200), (80, 200), (80, 21000), (110, 35000)])
def test_attention_nan(hip, M, Lmax):
    """A NaN that a row sees makes that row NaN (a value's: in its group of 64 dimensions); one that it does not
    see leaves every bit of it."""
    B, H, Hkv, hd, n = 2, 4, 2, 128, 180
    q, k, v = _inputs(M, B, n, H, Hkv, hd)
    q = q[:, :M]
    pos = [n - M, 60]
    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, n, k=k, v=v)
    clean = hip.kv4_attention(*_cuda(q), cache, _pos(pos), max_len=Lmax).cpu().numpy()
    assert np.isfinite(clean).all()
    kk, vv = k.copy(), v.copy()
    at = 60 + M // 2  # the middle row of sequence 1 is the first that sees it
    kk[1, at, 0, 3] = np.nan
    vv[1, at, 1, 70] = np.inf
    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, n, k=kk, v=vv)
    y = hip.kv4_attention(*_cuda(q), cache, _pos(pos), max_len=Lmax).cpu().numpy()
    want = clean.copy()
    want[1, M // 2:, :2] = np.nan
    want[1, M // 2:, 2:, 64:] = np.nan
    assert _same(y, want)


@pytest.mark.parametrize("M,Lmax", [(20, 100), (20, 42000), (128, 400000)])
def test_attention_nan_query(hip, M, Lmax):
    B, H, Hkv, hd, n = 1, 4, 2, 64, 70 + M
    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, n)
    q, _, _ = _inputs(6, B, M, H, Hkv, hd)
    clean = hip.kv4_attention(*_cuda(q), cache, _pos([70]), max_len=Lmax).cpu().numpy()
    q[0, 3, 1, 5], q[0, 7, 2, 9] = np.nan, np.inf
    y = hip.kv4_attention(*_cuda(q), cache, _pos([70]), max_len=Lmax).cpu().numpy()
    want = clean.copy()
    want[0, 3, 1] = want[0, 7, 2] = np.nan
    assert _same(y, want)


def test_strided_and_odd_inputs(hip):
    """Views: heads cut from a fused projection, every other sequence, an address that is not 16-byte aligned."""
    import torch

    B, M, H, Hkv, hd, Lmax = 2, 5, 4, 2, 64, 100
    q, k, v = _cuda(*_inputs(8, B, M, H, Hkv, hd))
    (rope,) = _cuda(_rope(Lmax, hd))
    a, b = hip.kv4_cache(Hkv, hd, Lmax, batch=B).zero_(), hip.kv4_cache(Hkv, hd, Lmax, batch=B).zero_()
    y = hip.kv4_append(q, k, v, a, rope, _pos([3, 80]))
    fused = torch.cat([q, k, v], 2)
    odd = torch.empty(rope.numel() + 1, device="cuda")[1:].view(rope.shape).copy_(rope)
    z = hip.kv4_append(fused[:, :, :H], fused[:, :, H:H + Hkv], fused[:, :, H + Hkv:], b, odd, _pos([3, 80]))
    assert torch.equal(y, z) and torch.equal(a, b)
    assert torch.equal(hip.kv4_attention(y, a, _pos([3, 80])), hip.kv4_attention(fused.copy_(torch.cat([y, k, v], 2))[:, :, :H], a, _pos([3, 80])))
    # q rotated in place
    hip.kv4_append(q, k, v, b, rope, _pos([3, 80]), q_out=q)
    assert torch.equal(q, y)


@pytest.mark.parametrize("B,M,H,Hkv,hd,Lmax", [(2, 1, 20, 5, 128, 300), (1, 1, 20, 5, 128, 4000), (2, 45, 8, 2, 64, 300),
                                               (2, 64, 8, 2, 128, 26000)])
def test_attention_in_place(hip, B, M, H, Hkv, hd, Lmax):
    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, 200)
    (q,) = _cuda(_inputs(6, B, M, H, Hkv, hd)[0])
    pos = _pos([200 - M, 120][:B])
    want = hip.kv4_attention(q, cache, pos, max_len=Lmax)
    assert hip.kv4_attention(q, cache, pos, max_len=Lmax, out=q) is q
    assert (q == want).all()


# (B, H, Hkv, hd, Lmax, positions): the token in a block's first and last place, outside the cache, in each wave's
# part and each split; 4, 8 and 16 rows a head, part of them; splits by length
STEPS = [
    (1, 20, 5, 128, 640, [0]), (1, 20, 5, 128, 640, [63]), (1, 20, 5, 128, 640, [64]), (1, 20, 5, 128, 640, [639]),
    (1, 20, 5, 128, 4000, [1537]), (1, 20, 5, 128, 4000, [70]), (2, 3, 3, 64, 130, [129, 31]),
    (4, 12, 12, 64, 777, [776, 5, 128, 400]), (3, 16, 1, 128, 300, [299, 0, 150]), (2, 16, 1, 64, 1500, [299, 1499]),
    (2, 14, 2, 64, 200, [100, 197]), (2, 14, 2, 128, 2000, [100, 1997]), (1, 30, 2, 128, 2000, [1000]), (1, 16, 1, 128, 1200, [1150]), (3, 24, 2, 64, 1100, [-3, 1099, 200]),
    (3, 4, 2, 64, 64, [-1, 63, 2147483647]), (5, 20, 5, 128, 3000, [2999, 0, 1200, 64, -1]),
    (64, 4, 2, 64, 2048, [(i * 997) % 2048 for i in range(64)]), (2, 5, 1, 128, 64, [-2, 64]),
]


@pytest.mark.parametrize("B,H,Hkv,hd,Lmax,pos", STEPS)
def test_step(hip, B, H, Hkv, hd, Lmax, pos):
    """One launch for both: the same bytes in the cache, the same outputs, over several steps."""
    import torch

    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, Lmax)
    mine = cache.clone()
    (rope,) = _cuda(_rope(Lmax, hd))
    at = _pos(pos)
    for i in range(3):
        q, k, v = _cuda(*_inputs(20 + i, B, 1, H, Hkv, hd))
        if i == 1:  # a group that reads as NaN
            k[0, 0, 0, 1] = float("nan")
            v[-1, 0, -1, -1] = float("inf")
        keep = [x.clone() for x in (q, k, v)]
        y = hip.kv4_step(q, k, v, mine, rope, at, max_len=Lmax)
        assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(keep, (q, k, v)))
        want = hip.kv4_attention(hip.kv4_append(q, k, v, cache, rope, at, max_len=Lmax), cache, at, max_len=Lmax)
        assert torch.equal(mine, cache)
        assert _same(y.cpu().numpy(), want.cpu().numpy())
        assert hip.kv4_step(q, k, v, mine, rope, at, max_len=Lmax, out=q) is q
        assert _same(q.cpu().numpy(), want.cpu().numpy()) and torch.equal(mine, cache)
        at = at + 1


def test_past_four_gigabytes(hip):
    """The last sequence of a cache of more than 2^32 bytes."""
    import torch

    B, Hkv, hd, Lmax, H, n = 60, 4, 128, 131072, 8, 100
    cache = hip.kv4_cache(Hkv, hd, Lmax, batch=B)
    assert cache.numel() > 1 << 32
    q, k, v = _inputs(9, 1, n, H, Hkv, hd)
    table = _rope(Lmax, hd)
    pos = [-1000] * (B - 1) + [Lmax - n]
    big = [np.zeros((B, n, x.shape[2], hd), np.float32) for x in (q, k, v)]
    for x, y in zip(big, (q, k, v)):
        x[-1] = y[0]
    cache[-1].zero_()
    hip.kv4_append(*_cuda(*big), cache, *_cuda(table), _pos(pos))
    got = [x[-1].cpu().numpy() for x in hip.kv4_read(cache, _pos(pos), n)]
    rk = np.stack([K4.rope(k[0, m], table, Lmax - n + m) for m in range(n)])
    for x, y in zip(got, (rk, v[0])):
        assert _same(x, K4.held(y.transpose(1, 0, 2)))
    # attention of the last sequence within the batch and alone (other splits of its keys: 131072 of them, sums
    # of numbers that are mostly zero, so the two agree far within fp32's sqrt(131072) roundings, 2e-5)
    tq = torch.zeros((B, 2, H, hd), device="cuda")
    tq[-1] = torch.from_numpy(q[0, -2:])
    alone = hip.kv4_attention(tq[-1:], cache[-1:].clone(), _pos([Lmax - 2]))
    both = hip.kv4_attention(tq, cache, _pos([-1000] * (B - 1) + [Lmax - 2]))
    assert (both[:-1] == 0).all()
    assert alone.abs().max() > 1e-6
    assert torch.linalg.norm(both[-1] - alone[0]) <= 2e-5 * torch.linalg.norm(alone)


@pytest.mark.parametrize("M,Lmax", [(1, 400), (1, 5000), (20, 400), (20, 42000), (64, 42000)])
def test_graph_and_streams(hip, M, Lmax):
    """A step (append, attention, read) captured on a stream of its own and replayed with moving positions, with
    eager work between the replays."""
    import torch

    B, H, Hkv, hd, n = 2, 8, 2, 128, 200
    cache, _ = _filled(hip, 5, B, H, Hkv, hd, Lmax, n)
    mine = cache.clone()
    (rope,) = _cuda(_rope(Lmax, hd))
    q, k, v = _cuda(*_inputs(1, B, M, H, Hkv, hd))
    pos = _pos([n, 100])

    def step(c):
        r = hip.kv4_append(q, k, v, c, rope, pos, max_len=Lmax)
        return [r, hip.kv4_attention(r, c, pos, max_len=Lmax), *hip.kv4_read(c, pos, M, max_len=Lmax)]

    if M == 1:
        two = step

        def step(c):
            return [*two(c), hip.kv4_step(q, k, v, c, rope, pos, max_len=Lmax)]

    step(mine.clone())  # (first launches)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        g.capture_begin()
        out = step(mine)
        g.capture_end()
    hip._bind_stream()
    for i in range(4):
        for x, y in zip((q, k, v), _cuda(*_inputs(10 + i, B, M, H, Hkv, hd))):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        want = step(cache)
        for x, y in zip(out, want):
            assert torch.equal(x, y)
        assert torch.equal(cache, mine)
        pos += M
    torch.cuda.synchronize()


def test_prompt_then_steps(hip):
    """As a program uses them: a prompt in two chunks, then single tokens, for three sequences of different lengths;
    every output against 64 bits over what the cache held at that moment."""
    B, H, Hkv, hd, Lmax = 3, 8, 2, 64, 160
    table = _rope(Lmax, hd)
    (rope,) = _cuda(table)
    cache = hip.kv4_cache(Hkv, hd, Lmax, batch=B)
    pos = np.array([0, 7, 90], np.int32)
    held = [np.zeros((B, Hkv, Lmax, hd), np.float32) for _ in range(2)]
    # sequences 1 and 2 have a past
    _, k, v = _inputs(50, B, 90, H, Hkv, hd)
    past = _pos([-90, -83, 0])
    hip.kv4_append(*_cuda(np.zeros((B, 90, H, hd), np.float32), k, v), cache, rope, past)
    for b, p in enumerate([-90, -83, 0]):
        for m in range(90):
            if p + m >= 0:
                held[0][b, :, p + m], held[1][b, :, p + m] = K4.held(K4.rope(k[b, m], table, p + m)), K4.held(v[b, m])
    for step, M in enumerate([20, 30] + [1] * 6):
        q, k, v = _inputs(60 + step, B, M, H, Hkv, hd)
        tq = hip.kv4_append(*_cuda(q, k, v), cache, rope, _pos(pos))
        y = hip.kv4_attention(tq, cache, _pos(pos)).cpu().numpy()
        rq = np.zeros_like(q)
        for b in range(B):
            for m in range(M):
                p = int(pos[b]) + m
                rq[b, m] = K4.rope(q[b, m], table, p)
                held[0][b, :, p], held[1][b, :, p] = K4.held(K4.rope(k[b, m], table, p)), K4.held(v[b, m])
        want = K4.attention(rq, *held, pos)
        # (at most 156 keys: the derived bound's factor, on magnitudes that are at most 5 here)
        assert np.abs(y - want).max() <= (2 * (404 * 60 + 4) + 4 * 156 + 60) * 2.0 ** -24 * 5
        assert np.linalg.norm(y - want) <= 2e-6 * np.linalg.norm(want)
        pos += M
