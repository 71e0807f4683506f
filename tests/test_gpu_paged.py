"""The paged KV cache on the GPU against its definition in 64 bits (oracle/paged_oracle.py).

Tolerances, u = 2^-24 (half a step of fp32):
  rotated numbers   u |y|: products and difference in 64 bits, rounded once (and the 64 bits' own 2^-53 of the products)
  cached numbers    half a step of the cache's type on top of that (bf16 2^-8, fp16 2^-11 relative, or half its smallest
                    step 2^-25; fp32 none); values are equal to torch's rounding
  attention         products are exact or fp32 ones and all sums are fp32.  A score is a sum of hd products whose partial sums are
                    no more than A = sum |q k| / sqrt(hd): its error is taken as (16 + 2 sqrt(3 hd)) u A (two standard
                    deviations of 3 hd roundings, plus the scaling's), which shifts a weight by as much relative to itself; the sums over
                    n slots of weights and of weighted values come to (64 + 4 sqrt(n)) u of sum p |v| likewise, with the exponential's
                    own units.  Together (2 (16 + 2 sqrt(3 hd)) A + 64 + 4 sqrt(n)) u sum p |v|.
  weights           the same with a weight for the value, and an fp32 addition: u of the sum
"""
import math

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 0.0}


def rope_angles(rows, rotary, theta=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * theta ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64) / rotary)
    return torch.stack([a.cos(), a.sin()], -1).float()


def make(lens, Hkv=2, hd=64, page=16, dtype="bf16", spare=3, extra=0, seed=0, scale=1.0):
    """(cache, table, lens) on the CPU: pages shuffled, `extra` more slots a sequence, what is not held NaN."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-(max(n, 0) + extra) // page) for n in lens]
    P = max(1, max(need))
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((len(lens), P), -1, dtype=torch.int32)
    cache = torch.full((2, pages, Hkv, page, hd), math.nan, dtype=TYPES[dtype])
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for t in range(0, max(lens[b], 0), page):
            m = min(page, lens[b] - t)
            cache[:, table[b, t // page].long(), :, :m] = (torch.randn((2, Hkv, m, hd), generator=gen) * scale).to(cache.dtype)
    return cache, table, torch.tensor(lens, dtype=torch.int32)


def attention_bound(o, size, most, lens):
    hd, n = o.shape[-1], lens.clamp(min=1).double().view(-1, 1, 1, 1)
    return (2 * (16 + 2 * math.sqrt(3 * hd)) * most + 64 + 4 * n.sqrt()) * U * size + 2.0 ** -126


def check_attention(hip, cache, table, lens, q, weights=None, call=None):
    o, w, size, most = PO.attend(q, cache, table, lens)
    dev = lambda x: x.cuda()  # noqa: E731
    wd = weights.cuda() if weights is not None else None
    got = call(wd) if call else hip.paged_attention(dev(q), dev(cache), dev(table), dev(lens), weights=wd)
    bound = attention_bound(o, size, most, lens)
    err = (got.cpu().double() - o).abs()
    assert (err <= bound).all(), f"off by {(err / bound).max().item()} times the bound"
    if weights is not None:
        S = w.shape[2]
        n = lens.clamp(min=1).double().view(-1, 1, 1)
        A = most.amax((1, 2, 3)).view(-1, 1, 1)
        want = weights[:, :, :S].double() + w
        bound = (2 * (16 + 2 * math.sqrt(3 * q.shape[-1])) * A + 64 + 4 * n.sqrt()) * U * w + U * want.abs() + 2.0 ** -126
        wc = wd.cpu()
        assert ((wc[:, :, :S].double() - want).abs() <= bound).all()
        assert torch.equal(wc[:, :, :S][w == 0], weights[:, :, :S][w == 0])  # slots not attended to
        assert torch.equal(wc[:, :, S:], weights[:, :, S:])
    return got


# ---- append ------------------------------------------------------------------------------


def append_case(hip, lens, M, H, Hkv, hd, page, dtype, rotary, interleaved, ahead=0, counts=None, in_place=False, seed=1):
    cache, table, lens = make(lens, Hkv, hd, page, dtype, extra=M, seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    B = len(lens)
    q, k, v = (torch.randn((B, M, n, hd), generator=gen) * 3 for n in (H, Hkv, Hkv))
    rope = rope_angles(int(lens.max()) + ahead + M + 1, rotary)
    pos = lens + ahead
    if counts is not None:
        counts = torch.tensor(counts, dtype=torch.int32)
    want_q, rows = PO.append(q, k, v, cache, table, lens, rope, pos, counts, interleaved)
    c, qd = cache.cuda(), q.cuda()
    got = hip.paged_append(qd, k.cuda(), v.cuda(), c, table.cuda(), lens.cuda(), rope.cuda(), pos.cuda(),
                           counts=counts.cuda() if counts is not None else None, interleaved=interleaved, q_out=qd if in_place else None)
    assert not in_place or got is qd
    assert ((got.cpu().double() - want_q).abs() <= U * want_q.abs() + 2.0 ** -46).all()
    c = c.cpu()
    written = torch.zeros(cache.shape[1], page, dtype=torch.bool)
    for (n, r), (key, value) in rows.items():
        written[n, r] = True
        bound = (HALF[dtype] * (1 + U) + U) * key.abs() + 2.0 ** -25
        assert ((c[0, n, :, r].double() - key).abs() <= bound).all()
        assert torch.equal(c[1, n, :, r], value.to(cache.dtype))
    assert int(written.sum()) == len(rows)
    left = ~written[None, :, None, :, None].expand_as(cache)
    assert torch.equal(torch.nan_to_num(c[left].float(), 7.0), torch.nan_to_num(cache[left].float(), 7.0))  # the rest as it was


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,rotary", [(64, 64), (64, 16), (64, 24), (128, 128), (128, 8), (128, 120)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(hip, dtype, hd, rotary, interleaved):
    append_case(hip, [0, 5, 40], 3, 6, 2, hd, 16, dtype, rotary, interleaved)


@pytest.mark.parametrize("lens,M,H,Hkv,page,kw", [
    ([0], 1, 1, 1, 16, {}), ([15], 1, 20, 5, 16, {}), ([16], 2, 4, 4, 16, {}), ([63, 64, 65, 1], 70, 7, 1, 64, {}),
    ([300], 257, 8, 2, 256, {}), ([7, 100], 33, 16, 2, 32, dict(ahead=1000)), ([3, 9, 30], 20, 3, 3, 128, dict(counts=[20, 0, 7])),
    ([3, 9], 5, 3, 3, 16, dict(counts=[9, -1])), ([11, 20], 6, 8, 2, 16, dict(in_place=True)),
    ([2] * 37, 1, 5, 5, 16, dict(in_place=True))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_shapes(hip, lens, M, H, Hkv, page, kw, interleaved):
    append_case(hip, lens, M, H, Hkv, 128, page, "bf16", 64, interleaved, **kw)


def test_append_without_a_place(hip):
    """Holes, slots and positions outside: nothing is written, their q is 0."""
    cache, table, lens = make([0, 0, 0, 0, 0], extra=32)
    table[1, 0], table[2, 1], table[3, 0] = -1, cache.shape[1], 2 ** 31 - 1
    lens = torch.tensor([30, 10, 10, -5, 2 ** 31 - 2], dtype=torch.int32)
    pos = torch.tensor([0, -2, 3, 4, 5], dtype=torch.int32)
    q, k, v = torch.randn(5, 9, 4, 64), torch.randn(5, 9, 2, 64), torch.randn(5, 9, 2, 64)
    rope = rope_angles(10, 64)
    want, rows = PO.append(q, k, v, cache, table, lens, rope, pos)
    c = cache.cuda()
    got = hip.paged_append(*(x.cuda() for x in (q, k, v)), c, table.cuda(), lens.cuda(), rope.cuda(), pos.cuda()).cpu()
    assert torch.equal(got == 0, want == 0) and (want == 0).any() and (want != 0).any()
    assert int((~c.isnan()).any(-1).sum()) == 2 * 2 * len(rows)


def test_append_rounds_to_nearest_even(hip):
    """Ties, overflow and subnormals of the cache's type."""
    x = torch.zeros(1, 1, 1, 64)
    x[0, 0, 0, :12] = torch.tensor([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 65519.0, 65520.0, -7e4, 2.0 ** -25,
                                    3 * 2.0 ** -25, 2.0 ** -130, 3.39e38, -0.0])
    for dtype in TYPES:
        cache, table, lens = make([0], 1, extra=1, dtype=dtype)
        c = cache.cuda()
        hip.paged_append(torch.ones(1, 1, 1, 64).cuda(), x.cuda(), x.cuda(), c, table.cuda(), lens.cuda(), rope_angles(1, 64).cuda(), lens.cuda())
        n = int(table[0, 0])
        assert torch.equal(c[1, n, 0, 0].cpu(), x.view(64).to(TYPES[dtype]))
        assert torch.equal(c[0, n, 0, 0].cpu(), x.view(64).to(TYPES[dtype]))  # (position 0: no turn)


def test_append_cancelling_pairs(hip):
    """x cos - y sin where the products agree to the last bits: still within the bound."""
    rope = torch.tensor([[[0.6, 0.8]] * 32]).float()
    q = torch.full((1, 1, 2, 64), 0.8) + torch.randn(1, 1, 2, 64) * 2.0 ** -20
    q[..., 32:] = 0.6
    cache, table, lens = make([0], 2, extra=1)
    want, _ = PO.append(q, q, q, cache, table, lens, rope, lens)
    got = hip.paged_append(q.cuda(), q.cuda(), q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), rope.cuda(), lens.cuda()).cpu()
    assert ((got.double() - want).abs() <= U * want.abs() + 2.0 ** -52).all()


# ---- attention ---------------------------------------------------------------------------


def queries(lens, H, hd, seed=5, scale=1.5):
    return torch.randn((len(lens), 1, H, hd), generator=torch.Generator().manual_seed(seed)) * scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (20, 5), (21, 3), (16, 1), (34, 2)])
def test_attention(hip, dtype, hd, page, H, Hkv):
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 64, 130, 517]
    cache, table, n = make(lens, Hkv, hd, page, dtype)
    check_attention(hip, cache, table, n, queries(lens, H, hd))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [40], [2500], [3000, 10, 0, 1200], [700] * 9])
@pytest.mark.parametrize("H,Hkv,hd", [(20, 5, 128), (6, 6, 64), (40, 2, 64)])
def test_attention_weights(hip, dtype, lens, H, Hkv, hd):
    cache, table, n = make(lens, Hkv, hd, 32, dtype, seed=len(lens))
    start = torch.rand((len(lens), Hkv, table.shape[1] * 32 + 5), generator=torch.Generator().manual_seed(3))
    check_attention(hip, cache, table, n, queries(lens, H, hd), weights=start)


def test_attention_long(hip):
    """Many splits, more than 64 tiles a wave's table look-up, sequences far apart in length."""
    for B, page, dtype in ((1, 64, "bf16"), (3, 16, "fp16"), (40, 256, "bf16")):
        lens = [40000] + [1 + 97 * b for b in range(B - 1)]
        cache, table, n = make(lens, 1, 64, page, dtype)
        check_attention(hip, cache, table, n, queries(lens, 3, 64), weights=torch.zeros(B, 1, table.shape[1] * page))


def test_attention_many_heads_long(hip):
    """One split a head (as many heads as fill the GPU), more than 64 tiles a wave."""
    lens = [9000] + [3] * 255
    cache, table, n = make(lens, 4, 64, 16, "bf16")
    check_attention(hip, cache, table, n, queries(lens, 4, 64))


def test_attention_large_batches(hip):
    """More sequences than lanes, and than a launch has places to cut them for; more heads than a workgroup's tile."""
    gen = torch.Generator().manual_seed(12)
    lens = torch.randint(0, 600, (130,), generator=gen).tolist() + [3000]
    cache, table, n = make(lens, 2, 64, 32, "bf16")
    check_attention(hip, cache, table, n, queries(lens, 4, 64), weights=torch.zeros(131, 2, table.shape[1] * 32))
    lens = torch.randint(0, 20, (4200,), generator=gen).tolist() + [300]
    cache, table, n = make(lens, 1, 64, 16, "fp16")
    check_attention(hip, cache, table, n, queries(lens, 1, 64))
    check_attention(hip, cache, table, n, queries(lens, 1, 64), weights=torch.zeros(4201, 1, table.shape[1] * 16))
    for B, Hkv in ((60, 10), (300, 2)):  # (more heads than run at once, one sequence far longer than the others)
        lens = torch.randint(0, 40, (B,), generator=gen).tolist()
        lens[B // 3], lens[-1] = 6000, 1500
        cache, table, n = make(lens, Hkv, 64, 32, "bf16")
        check_attention(hip, cache, table, n, queries(lens, Hkv, 64), weights=torch.zeros(B, Hkv, table.shape[1] * 32))
    lens = [900, 40]
    cache, table, n = make(lens, 1, 64, 16, "bf16")
    check_attention(hip, cache, table, n, queries(lens, 1024, 64), weights=torch.zeros(2, 1, table.shape[1] * 16))


def test_attention_table_much_longer_than_needed(hip):
    """A table for 2^20 slots over sequences that hold a few."""
    lens = [70, 0, 1300]
    for dtype in TYPES:
        cache, table, n = make(lens, 2, 64, 64, dtype)
        wide = torch.full((3, 1 << 14), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        q = queries(lens, 8, 64)
        got = check_attention(hip, cache, wide, n, q)
        start = torch.zeros(3, 2, 1 << 20)
        w = start.cuda()
        o, sums, size, most = PO.attend(q, cache, table, n)
        again = hip.paged_attention(q.cuda(), cache.cuda(), wide.cuda(), n.cuda(), weights=w)
        assert ((again.cpu().double() - o).abs() <= attention_bound(o, size, most, n)).all() and (w[:, :, 1344:] == 0).all()
        assert ((w[:, :, :1344].cpu().double() - sums).abs() <= 1e-5 * sums + 1e-30).all() and torch.allclose(got, again, atol=1e-5)


def test_attention_workspace_holds_anything(hip):
    """The same workspace, whatever is in it: noise, ones, the words of the calls before, other shapes'."""
    from rotor import _hip

    cases = []
    for lens, H, Hkv, hd in (([1500], 20, 5, 128), ([900, 200], 8, 2, 64), ([300] * 7, 12, 12, 64)):
        cache, table, n = make(lens, Hkv, hd, 64, "bf16")
        q = queries(lens, H, hd)
        o, _, size, most = PO.attend(q, cache, table, n)
        bound = attention_bound(o, size, most, n)
        c, t, m = cache.cuda(), table.cuda(), n.cuda()
        rows = Hkv * 64 * hd
        pages = _hip.PAGES.pack(c.data_ptr(), c.stride(0), rows, t.data_ptr(), m.data_ptr(), _hip.PAGED_BF16, c.shape[1], Hkv, 64, hd, len(lens), t.shape[1])
        cases.append((pages, q.cuda(), H, o, bound, (c, t, m)))
    need = max(hip.lib.rt_paged_attention_workspace(c[0], c[2], 0) for c in cases)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    fills = [lambda: ws.fill_(255), lambda: ws.random_(0, 256), lambda: ws.zero_()] + [lambda: None] * 6
    hip._bind_stream()
    for fill in fills:
        fill()
        for pages, q, H, o, bound, _ in cases:
            outs = [torch.empty_like(q) for _ in range(2)]
            for out in outs:  # (one behind the other, nothing waits)
                _hip.check(hip.lib.rt_paged_attention(hip.ctx, pages, q.data_ptr(), H, None, 0, out.data_ptr(), ws.data_ptr(), need))
            assert ((outs[0].cpu().double() - o).abs() <= bound).all() and torch.equal(outs[0], outs[1])


def test_attention_on_two_streams(hip):
    """Calls that run at the same time."""
    cache, table, n = make([1500, 700], 5, 128, 64, "bf16")
    q = queries([0] * 2, 20, 128).cuda()
    c, t, m = cache.cuda(), table.cuda(), n.cuda()
    want = hip.paged_attention(q, c, t, m)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(hip.paged_attention(q, c, t, m))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,H,Hkv,hd", [
    ([1024], 4, 1, 64), ([1025], 4, 1, 64), ([1024, 0, 513, 1], 8, 2, 128), ([256, 256], 16, 1, 128), ([288], 16, 1, 64), ([32] * 70, 17, 1, 64),
    ([500] * 16, 15, 3, 64), ([31 + b for b in range(90)], 6, 6, 64), ([576, 40], 14, 2, 64)])
def test_attention_weights_of_short_caches(hip, dtype, lens, H, Hkv, hd):
    """As long as one launch adds them up, and longer; three calls onto the same sums."""
    cache, table, n = make(lens, Hkv, hd, 32, dtype, seed=H)
    start = torch.rand((len(lens), Hkv, table.shape[1] * 32 + 3), generator=torch.Generator().manual_seed(4))
    q = queries(lens, H, hd)
    want = check_attention(hip, cache, table, n, q, weights=start)
    w, c, t, m = start.cuda(), cache.cuda(), table.cuda(), n.cuda()
    outs = [hip.paged_attention(q.cuda(), c, t, m, weights=w) for _ in range(3)]
    assert all(torch.equal(o, want) for o in outs)
    check_attention(hip, cache, table, n, q)  # (without weights pieces may be joined in another order: each within its bound)
    sums = PO.attend(q, cache, table, n)[1]
    S = sums.shape[2]
    total = start[:, :, :S].double() + 3 * sums
    # each time as near as one call's, and an addition's rounding
    most = PO.attend(q, cache, table, n)[3].amax((1, 2, 3)).view(-1, 1, 1)
    share = 2 * (16 + 2 * math.sqrt(3 * hd)) * most + 64 + 4 * n.clamp(min=1).double().sqrt().view(-1, 1, 1)
    assert ((w[:, :, :S].cpu().double() - total).abs() <= 3 * U * (share * sums + total) + 2.0 ** -126).all()


def test_attention_weights_on_streams(hip):
    """Calls that run at the same time, each with sums of its own, in workspaces that hold anything."""
    cache, table, n = make([900, 300], 5, 128, 64, "bf16")
    q = queries([0] * 2, 20, 128).cuda()
    c, t, m = cache.cuda(), table.cuda(), n.cuda()
    want = torch.zeros(2, 5, t.shape[1] * 64, device="cuda")
    out = hip.paged_attention(q, c, t, m, weights=want)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                torch.full((1 << 20,), -1 - i, dtype=torch.int32, device="cuda")  # (what the next workspace holds)
                w = torch.zeros_like(want)
                got.append((hip.paged_attention(q, c, t, m, weights=w), w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) and torch.equal(w, want) for o, w in got)


def test_attention_holes(hip):
    """Holes in the middle and at the end, whole sequences of them; lengths past the table and below 0."""
    lens = [200, 64, 90, 128, 40]
    cache, table, _ = make(lens, 2, 64, 16, "bf16", extra=16)
    table[0, 3], table[0, 7], table[1], table[2, :5], table[3, 7] = -1, cache.shape[1] + 5, -3, 2 ** 31 - 1, -2 ** 31
    n = torch.tensor([200, 64, 90, 128, -1], dtype=torch.int32)
    start = torch.rand(5, 2, table.shape[1] * 16)
    got = check_attention(hip, cache, table, n, queries(lens, 8, 64), weights=start)
    assert (got[1] == 0).all() and (got[4] == 0).all()
    cache, table, _ = make([160, 160], 2, 64, 32, "fp32")
    n = torch.tensor([10 ** 9, 160], dtype=torch.int32)
    check_attention(hip, cache, table, n, queries([1, 1], 4, 64))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_what_is_not_held(hip, dtype):
    """Slots past the length hold infinities and NaN, in the last tile, in the page and in other pages: no trace of them."""
    cache, table, n = make([70, 5, 33], 2, 128, 64, dtype, seed=9)
    other = cache.clone()
    other[other.isnan()] = math.inf
    low = cache.clone()
    low[low.isnan()] = torch.finfo(low.dtype).min
    q = queries([0] * 3, 10, 128).cuda()
    outs = [hip.paged_attention(q, c.cuda(), table.cuda(), n.cuda()) for c in (cache, other, low)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(hip, dtype):
    """Scores of thousands: one slot takes it all, wherever it lies; and scores far below zero."""
    for seed in range(3):
        cache, table, n = make([300, 77], 2, 64, 32, dtype, seed=seed, scale=8.0)
        check_attention(hip, cache, table, n, queries([0] * 2, 6, 64, seed=seed, scale=60.0))
    cache, table, n = make([90], 1, 64, 32, dtype, scale=1.0)
    cache[0] = cache[0].abs()
    check_attention(hip, cache, table, n, -queries([0], 3, 64).abs() * 50)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_numbers_of_very_different_sizes(hip, dtype):
    """Values 2^20 apart under weights 2^-20 apart, and queries and keys whose dimensions are: every bit counts."""
    cache, table, n = make([64], 1, 64, 32, dtype, seed=4)
    pages = table[0].long()
    x = cache[:, pages].clone()  # [2, P, 1, 32, 64]
    x[0, ..., 0] = 0
    x[0, 0, 0, 3, 0] = 16.0      # this key's score is 16 * q0 / 8 above the others'
    x[1, 0, 0, 3] = 2.0 ** -10   # and its value small
    x[1, 1, 0, 5] = 2.0 ** 14    # a value of weight 2^-20 that is large
    cache[:, pages] = x
    q = torch.full((1, 1, 2, 64), 2.0 ** -9)
    q[..., 0] = 20 * math.log(2) / 2
    check_attention(hip, cache, table, n, q)
    cache, table, n = make([64], 1, 64, 32, dtype, seed=6)
    x = cache[0, table[0].long()]
    x[..., :32] *= 2.0 ** -9
    x[..., 32:] *= 2.0 ** 5
    cache[0, table[0].long()] = x
    q = queries([0], 2, 64)
    q[..., :32] *= 2.0 ** 9
    q[..., 32:] *= 2.0 ** -7
    check_attention(hip, cache, table, n, q)


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 40])
def test_attention_queries_and_keys_of_any_size(hip, scale):
    for dtype in ("bf16", "fp32"):
        cache, table, n = make([100], 2, 64, 32, dtype, seed=7)
        cache[0] = (cache[0].float() * scale).to(cache.dtype)
        check_attention(hip, cache, table, n, queries([0], 4, 64) / scale)
    cache, table, n = make([100], 2, 64, 32, "fp16", seed=7)
    cache[0] = (cache[0].float() * 2.0 ** -12).to(cache.dtype)
    check_attention(hip, cache, table, n, queries([0], 4, 64) * 2.0 ** 12)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_not_finite(hip, dtype):
    """A held key, value or query that is not finite shows in its own heads' outputs and nowhere else."""
    cache, table, n = make([50, 50], 2, 64, 32, dtype)
    q = queries([0] * 2, 4, 64)
    good = hip.paged_attention(q.cuda(), cache.cuda(), table.cuda(), n.cuda())
    for bad in (math.nan, math.inf, -math.inf):
        c = cache.clone()
        c[0, table[0, 1].long(), 1, 3, 5] = bad
        out = hip.paged_attention(q.cuda(), c.cuda(), table.cuda(), n.cuda())
        same = torch.ones_like(good, dtype=torch.bool)
        same[0, :, 2:] = False
        assert torch.equal(out[same], good[same])
        if math.isnan(bad):
            assert out[0, :, 2:].isnan().all()
        c = cache.clone()
        c[1, table[1, 0].long(), 0, 7, 9] = bad
        out = hip.paged_attention(q.cuda(), c.cuda(), table.cuda(), n.cuda())
        same = torch.ones_like(good, dtype=torch.bool)
        same[1, :, :2, 9] = False
        assert torch.equal(out[same], good[same]) and not out[1, :, :2, 9].isfinite().any()
        x = q.clone()
        x[1, 0, 3, 11] = bad
        out = hip.paged_attention(x.cuda(), cache.cuda(), table.cuda(), n.cuda())
        same = torch.ones_like(good, dtype=torch.bool)
        same[1, 0, 3] = False
        assert torch.equal(out[same], good[same])
        if math.isnan(bad):
            assert out[1, 0, 3].isnan().all()


def test_attention_in_place_and_layouts(hip):
    """out = q; layers of one larger tensor; keys next to values; other types and strides of q; shared pages."""
    cache, table, n = make([90, 40], 2, 64, 32, "bf16")
    q = queries([0] * 2, 8, 64)
    want = hip.paged_attention(q.cuda(), cache.cuda(), table.cuda(), n.cuda())
    x = q.cuda()
    assert hip.paged_attention(x, cache.cuda(), table.cuda(), n.cuda(), out=x) is x and torch.equal(x, want)
    layers = torch.zeros((cache.shape[1], 3, 2, *cache.shape[2:]), dtype=cache.dtype, device="cuda")
    layers[:, 1] = cache.cuda().transpose(0, 1)
    assert torch.equal(hip.paged_attention(q.cuda(), layers[:, 1].transpose(0, 1), table.cuda(), n.cuda()), want)
    wide = torch.zeros(2, 1, 8, 128, device="cuda")
    wide[..., 1:65] = q.cuda()
    assert torch.equal(hip.paged_attention(wide[..., 1:65], cache.cuda(), table.cuda(), n.cuda()), want)
    assert torch.equal(hip.paged_attention(q.double().cuda(), cache.cuda(), table.cuda(), n.cuda()), want)
    shared = torch.stack([table[0], table[0]])
    m = torch.tensor([90, 61], dtype=torch.int32)
    check_attention(hip, cache, shared, m, q)


def test_cache_past_32_bits(hip):
    """Pages whose offsets pass 2^32 bytes and 2^31 elements."""
    pages, page, hd = 40000, 256, 128
    cache = torch.zeros((2, pages, 1, page, hd), dtype=torch.bfloat16, device="cuda")  # 5.2 GB: elements past 2^31
    table = torch.tensor([[pages - 1, 0, 17000], [33000, 1, pages - 2]], dtype=torch.int32)
    n = torch.tensor([520, 700], dtype=torch.int32)
    small = torch.zeros((2, 6, 1, page, hd), dtype=torch.bfloat16)
    small[:] = torch.randn(small.shape, generator=torch.Generator().manual_seed(1))
    cache[:, table.flatten().long().cuda()] = small.cuda()
    near = torch.arange(6, dtype=torch.int32).view(2, 3)
    q = queries([0] * 2, 4, hd).cuda()
    assert torch.equal(hip.paged_attention(q, cache, table.cuda(), n.cuda()), hip.paged_attention(q, small.cuda(), near.cuda(), n.cuda()))
    k = torch.randn(2, 1, 1, hd, device="cuda")
    rope = rope_angles(701, hd).cuda()
    hip.paged_append(q, k, k, cache, table.cuda(), n.cuda(), rope, n.cuda())
    assert torch.equal(cache[1, pages - 1 if 520 < 256 else 17000, 0, 520 % 256], k[0, 0, 0].bfloat16())
    assert torch.equal(cache[1, pages - 2, 0, 700 % 256], k[1, 0, 0].bfloat16())
    fresh = torch.tensor([[pages - 3], [39000]], dtype=torch.int32).cuda()
    w = torch.rand(2, 1, 768, device="cuda")
    kept, m, _ = hip.paged_evict(cache, table.cuda(), n.cuda(), w, 100, 10, fresh)
    for b in range(2):
        t = kept[b, 0].long()
        assert torch.equal(cache[:, fresh[b, 0].long(), 0, :100], cache[:, table[b].cuda()[t // 256].long(), 0, t % 256])


# ---- step --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,hd,rotary,interleaved", [(20, 5, 128, 128, False), (6, 6, 64, 64, True), (34, 2, 64, 24, False), (4, 1, 128, 8, True)])
@pytest.mark.parametrize("lens,page", [([0, 1, 15, 16, 31, 32, 200], 16), ([63, 64, 2000], 64), ([255, 256, 3, 511, 40], 256)])
def test_step(hip, dtype, H, Hkv, hd, rotary, interleaved, lens, page):
    """The same numbers in the cache as paged_append leaves, and attention over them."""
    cache, table, n = make(lens, Hkv, hd, page, dtype, extra=1)
    gen = torch.Generator().manual_seed(8)
    B = len(lens)
    q, k, v = (torch.randn((B, 1, m, hd), generator=gen) for m in (H, Hkv, Hkv))
    rope, pos = rope_angles(max(lens) + 12, rotary), n + 11
    one, two = cache.cuda(), cache.cuda()
    turned = hip.paged_append(*(x.cuda() for x in (q, k, v)), one, table.cuda(), n.cuda(), rope.cuda(), pos.cuda(), interleaved=interleaved)
    start = torch.rand((B, Hkv, table.shape[1] * page), generator=gen)
    args = [x.cuda() for x in (q, k, v)] + [two, table.cuda(), n.cuda(), rope.cuda(), pos.cuda()]
    check_attention(hip, one.cpu(), table, n + 1, turned.cpu(), weights=start,
                    call=lambda w: hip.paged_step(*args, interleaved=interleaved, weights=w))
    bits = torch.int32 if dtype == "fp32" else torch.int16
    assert torch.equal(one.view(bits), two.view(bits))
    again = hip.paged_step(*args, interleaved=interleaved, out=args[0])
    assert again is args[0] and torch.equal(again, hip.paged_attention(turned, one, table.cuda(), n.cuda() + 1))


def test_step_without_a_place(hip):
    """No slot, no page, no angle: nothing written, zeros, and the others as they would be."""
    cache, table, _ = make([40] * 6, extra=8)
    table[1, 2] = -1
    lens = torch.tensor([40, 40, 48, -1, 40, 40], dtype=torch.int32)
    pos = torch.tensor([40, 40, 40, 40, 50, -1], dtype=torch.int32)
    q, k, v = torch.randn(6, 1, 4, 64), torch.randn(6, 1, 2, 64), torch.randn(6, 1, 2, 64)
    rope = rope_angles(50, 64)
    c, w = cache.cuda(), torch.zeros(6, 2, 48, device="cuda")
    out = hip.paged_step(*(x.cuda() for x in (q, k, v)), c, table.cuda(), lens.cuda(), rope.cuda(), pos.cuda(), weights=w)
    assert (out[1:] == 0).all() and (w[1:] == 0).all() and out[0].isfinite().all() and (out[0] != 0).all()
    changed = (c.cpu().float().nan_to_num(7.0) != cache.float().nan_to_num(7.0)).any(-1).nonzero()
    assert {(int(p), int(r)) for _, p, _, r in changed} == {(int(table[0, 2]), 8)}


# ---- evict -------------------------------------------------------------------------------


def check_evict(hip, cache, table, lens, weights, keep, recent, spare):
    """spare: pages for the new table (as many as B * ceil(keep / page))."""
    B, Hkv, _ = weights.shape
    page = cache.shape[3]
    want = PO.evict(cache, table, lens, weights, keep, recent)
    new = spare[torch.randperm(len(spare))[:B * -(-keep // page)]].view(B, -1).int()
    c = cache.cuda()
    kept, n, left = (x.cpu() for x in hip.paged_evict(c, table.cuda(), lens.cuda(), weights.cuda(), keep, recent, new.cuda()))
    c = c.cpu()
    expect = cache.clone()
    for b in range(B):
        assert int(n[b]) == len(want[b][0])
        for h in range(Hkv):
            t = torch.tensor(want[b][h], dtype=torch.long)
            i = torch.arange(len(t))
            assert torch.equal(kept[b, h, :len(t)].long(), t) and (kept[b, h, len(t):] == -1).all(), (b, h)
            assert torch.equal(left[b, h, :len(t)].nan_to_num(-7.0), weights[b, h, t].nan_to_num(-7.0)) and (left[b, h, len(t):] == 0).all()
            expect[:, new[b].long()[i // page], h, i % page] = cache[:, table[b].long()[t // page], h, t % page]
    bits = torch.int32 if cache.dtype == torch.float32 else torch.int16
    assert torch.equal(c.view(bits), expect.view(bits))
    return c, new, n, left


def evict_case(hip, lens, keep, recent, Hkv=2, hd=64, page=16, dtype="bf16", seed=0, weights=None):
    pages = len(lens) * -(-keep // page)
    cache, table, n = make(lens, Hkv, hd, page, dtype, spare=pages + 2, seed=seed)
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))
    gen = torch.Generator().manual_seed(seed + 1)
    w = torch.rand((len(lens), Hkv, table.shape[1] * page + 3), generator=gen) if weights is None else weights(gen, table.shape[1] * page)
    return check_evict(hip, cache, table, n, w, keep, recent, free)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,keep,recent,page", [
    ([1], 1, 0, 16), ([1], 1, 1, 16), ([0], 5, 2, 16), ([100], 1, 0, 16), ([100], 1, 1, 16), ([100], 50, 50, 32), ([100], 99, 7, 32),
    ([100, 3, 0, 64, 50], 50, 10, 64), ([64, 65, 63], 64, 0, 16), ([2500, 1100], 1024, 100, 256), ([5000, 40], 17, 3, 16)])
def test_evict(hip, dtype, hd, lens, keep, recent, page):
    evict_case(hip, lens, keep, recent, 3, hd, page, dtype)


def test_evict_ties_and_odd_weights(hip):
    """Equal weights in numbers, zeros of both signs, negative ones, infinities, NaN, neighbours in the last bit."""
    pick = lambda values: lambda gen, S: values[torch.randint(len(values), (3, 2, S), generator=gen)]  # noqa: E731
    inf, nan = math.inf, math.nan
    for values in ([0.0], [0.0, -0.0], [1.0, 2.0], [nan, 1.0, inf], [-inf, inf, -1.0, -2.0, 0.0], [-nan, nan, inf],
                   [1.0, 1.0 + 2.0 ** -23, 1.0 + 2.0 ** -22], [2.0 ** -149, 0.0, -2.0 ** -149, 2.0 ** -126]):
        values = torch.tensor(values)
        for keep, recent in ((1, 0), (40, 5), (170, 0), (299, 299)):
            evict_case(hip, [300, 171, 200], keep, recent, weights=pick(values), seed=keep)


def test_evict_holes(hip):
    """Slots in holes are never kept, recent or not; a new page in a hole is not written."""
    lens = [100, 100, 60, 100]
    cache, table, n = make(lens, 2, 64, 16, "bf16", spare=20)
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))
    table[0, 2], table[0, 6], table[1], table[3, 1:] = -1, 2 ** 31 - 1, -5, cache.shape[1]
    w = torch.rand(4, 2, table.shape[1] * 16)
    for keep, recent in ((30, 10), (30, 30), (64, 0)):
        check_evict(hip, cache, table, n, w, keep, recent, free)
    new = free[:8].view(4, 2).int()
    new[2, 0] = -1
    c = cache.cuda()
    kept, m, left = hip.paged_evict(c, table.cuda(), n.cuda(), w.cuda(), 20, 4, new.cuda())
    assert m.tolist() == [20, 0, 20, 16]
    t = kept[2, 0, 16:20].cpu().long()
    assert torch.equal(c[:, int(new[2, 1]), 0, :4].cpu(), cache[:, table[2].long()[t // 16], 0, t % 16])


def test_evict_long_ties_and_holes(hip):
    """Past 32768 slots: equal weights, odd ones, holes, everything kept and nothing but the recent."""
    inf, nan = math.inf, math.nan
    for values, keep, recent in (([0.0, 1.0], 20000, 0), ([nan, inf, -1.0, 0.0], 30000, 5000), ([1.0], 100, 100), ([2.0, 3.0], 34000, 33999)):
        values = torch.tensor(values)
        evict_case(hip, [33000, 40], keep, recent, 1, 64, 128,
                   weights=lambda gen, S: values[torch.randint(len(values), (2, 1, S), generator=gen)])
    cache, table, n = make([36000], 1, 64, 256, "bf16", spare=130)
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))
    table[0, 5:20], table[0, 130:] = -1, cache.shape[1]
    for keep, recent in ((32000, 4000), (33000, 0)):
        check_evict(hip, cache, table, n, torch.rand(1, 1, table.shape[1] * 256), keep, recent, free)


def test_evict_long(hip):
    evict_case(hip, [70000, 33000], 30000, 1000, 1, 64, 256)
    evict_case(hip, [40000], 1, 0, 1, 64, 256, weights=lambda gen, S: torch.ones(1, 1, S))


# ---- together ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_run_of_them(hip, dtype):
    """Two prompts of different lengths, steps that keep the weights, an eviction to fewer pages, steps on: against a plain
    cache in 64 bits that does the same."""
    B, H, Hkv, hd, page, keep, recent = 2, 8, 2, 64, 16, 40, 9
    gen = torch.Generator().manual_seed(11)
    cache = hip.paged_cache(Hkv, hd, 40, page, TYPES[dtype])
    order = torch.randperm(40, generator=gen).int()
    table, fresh = order[:14].view(B, 7).cuda(), order[14:24].view(B, 5).cuda()
    rope = rope_angles(200, 32)
    lens, pos = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    weights = torch.zeros(B, Hkv, 7 * page, device="cuda")
    counts = torch.tensor([60, 31], dtype=torch.int32)
    new = lambda M: [torch.randn((B, M, n, hd), generator=gen) for n in (H, Hkv, Hkv)]  # noqa: E731
    held = [[[], []] for _ in range(B)]  # keys and values [Hkv, hd] as the cache holds them

    def enter(k, v, b, m, p):
        held[b][0].append(PO.rotate(k[b, m].double(), rope[p], False).float().to(TYPES[dtype]).double())
        held[b][1].append(v[b, m].to(TYPES[dtype]).double())

    x = new(60)
    for b in range(B):
        for m in range(int(counts[b])):
            enter(x[1], x[2], b, m, m)
    hip.paged_append(*(t.cuda() for t in x), cache, table, lens, rope.cuda(), pos, counts=counts.cuda())
    lens += counts.cuda()
    pos += counts.cuda()
    sums = torch.zeros(B, Hkv, 7 * page, dtype=torch.float64)
    per_head = None
    for step in range(30):
        x = new(1)
        for b in range(B):
            enter(x[1], x[2], b, 0, int(pos[b]))
            if per_head is not None:
                for h in range(Hkv):
                    for i in range(2):
                        per_head[b][h][i].append(held[b][i][-1][h])
        out = hip.paged_step(*(t.cuda() for t in x), cache, table, lens, rope.cuda(), pos, weights=weights).cpu().double()
        for b in range(B):
            q = PO.rotate(x[0][b, 0].double(), rope[int(pos[b])], False)
            for h in range(H):
                kv = h // (H // Hkv)
                K, V = (torch.stack([r[kv] for r in held[b][i]]) for i in range(2)) if per_head is None else \
                    (torch.stack(per_head[b][kv][i]) for i in range(2))
                p = torch.softmax(K @ q[h] / hd ** 0.5, 0)
                sums[b, kv, :len(p)] += p
                # keys next to a border of bf16 may be rounded the other way: one step of one number in a few thousand
                # (a step 2^-7 of a key of up to 4, q up to 4, / 8, in a weight of at most 1, twice: 0.03 of it)
                tol = 1e-5 if dtype == "fp32" else 0.03
                assert (out[b, 0, h] - p @ V).abs().max() <= tol * (p @ V.abs()).max()
        lens += 1
        pos += 1
        if step == 14:
            n = lens.tolist()
            kept, lens, weights = hip.paged_evict(cache, table, lens, weights, keep, recent, fresh)
            assert lens.tolist() == [min(keep, m) for m in n]
            table = fresh
            per_head, old = [], sums
            sums = torch.zeros_like(sums)
            for b in range(B):
                per_head.append([])
                for h in range(Hkv):
                    t = kept[b, h, :int(lens[b])].tolist()
                    assert t == sorted(t) and t[-min(recent, len(t)):] == list(range(n[b] - min(recent, len(t)), n[b]))
                    lost = sorted(set(range(n[b])) - set(t))
                    if lost:
                        assert old[b, h, lost].max() <= old[b, h, t[:-recent]].min() * (1 + 1e-4) + 0.02 * (dtype != "fp32")
                    per_head[b].append([[held[b][i][s][h] for s in t] for i in range(2)])
                    sums[b, h, :len(t)] = old[b, h, t]
    tol = 1e-4 if dtype == "fp32" else 0.03
    assert ((weights.cpu().double() - sums).abs() <= tol * sums.clamp(min=1.0)).all()


def test_streams(hip):
    """Calls on a side stream, the next ones waiting for it by an event only."""
    cache, table, n = make([900, 300], 2, 64, 32, "bf16", extra=1)
    q, k = queries([0] * 2, 8, 64).cuda(), torch.randn(2, 1, 2, 64, device="cuda")
    rope = rope_angles(901, 64).cuda()
    c0, c1, t, m = cache.cuda(), cache.cuda(), table.cuda(), n.cuda()
    want = hip.paged_step(q, k, k, c0, t, m, rope, m)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        turned = hip.paged_append(q, k, k, c1, t, m, rope, m)
        got = hip.paged_attention(turned, c1, t, m + 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(c0.view(torch.int16), c1.view(torch.int16))


def test_graph(hip):
    """A captured step that advances by itself, and an eviction, replayed between eager work; two graphs alive at once."""
    cache, table, n = make([100, 30], 2, 64, 16, "bf16", extra=12, spare=12)
    q, k = queries([0] * 2, 8, 64).cuda(), torch.randn(2, 1, 2, 64, device="cuda")
    rope, t = rope_angles(120, 64).cuda(), table.cuda()
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))[:8].view(2, 4).int().cuda()

    def state():
        return [cache.cuda(), n.cuda(), torch.zeros(2, 2, t.shape[1] * 16, device="cuda")]

    def step(s):
        out = hip.paged_step(q, k, k, s[0], t, s[1], rope, s[1], weights=s[2])
        s[1] += 1
        return out

    a, b, e = state(), state(), state()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in (a, b):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(s)
                more = hip.paged_evict(s[0], t, s[1], s[2], 40, 5, free)
            graphs.append(g)
            outs.append((out, *more))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(6):
        want = (step(e), *hip.paged_evict(e[0], t, e[1], e[2], 40, 5, free))
        want = [x.clone() for x in want]
        torch.zeros(1 << 20, device="cuda").add_(1)
        for g in graphs:
            g.replay()
        for got in outs:
            assert all(torch.equal(x, y) for x, y in zip(got, want)), i
        torch.cuda.synchronize()
    assert torch.equal(a[0].view(torch.int16), e[0].view(torch.int16)) and torch.equal(b[2], e[2])


def test_the_same_twice(hip):
    """No order decides: the same call gives the same bits."""
    cache, table, n = make([3000, 1234, 10], 5, 128, 64, "bf16")
    q = queries([0] * 3, 20, 128).cuda()
    c, t, m = cache.cuda(), table.cuda(), n.cuda()
    runs = []
    for _ in range(3):
        w = torch.zeros(3, 5, t.shape[1] * 64, device="cuda")
        runs.append((hip.paged_attention(q, c, t, m, weights=w), w))
    for o, w in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(w, runs[0][1])


def test_model_with_scaled_angles(hip):
    """rope_scaling in a model's config reaches its angles: linear by 2 at even positions is plain at half of them."""
    import numpy as np

    from rotor.bitnet_model import BitNetModel, rope_table

    cfg = dict(vocab_size=512, d_model=512, n_layers=1, n_heads=4, n_kv_heads=2, d_ff=1024, max_seq_len=64, max_batch_tokens=32)
    rng = np.random.default_rng(3)
    p, state = "model.layers.0", {}
    for name, out, inner in (("self_attn.q_proj", 512, 512), ("self_attn.k_proj", 256, 512), ("self_attn.v_proj", 256, 512),
                             ("self_attn.o_proj", 512, 512), ("mlp.gate_proj", 1024, 512), ("mlp.up_proj", 1024, 512), ("mlp.down_proj", 512, 1024)):
        state[f"{p}.{name}.weight"] = rng.choice(np.array([0, 1, 2], np.uint8), (out, inner // 4, 4)) @ np.array([1, 4, 16, 64], np.uint8)
        state[f"{p}.{name}.weight_scale"] = np.array([0.02], np.float32)
    for name, size in (("input_layernorm", 512), ("post_attention_layernorm", 512), ("self_attn.attn_sub_norm", 512), ("mlp.ffn_sub_norm", 1024)):
        state[f"{p}.{name}.weight"] = np.ones(size, np.float32)
    state["model.norm.weight"] = np.ones(512, np.float32)
    state["model.embed_tokens.weight"] = torch.from_numpy(rng.standard_normal((512, 512)).astype(np.float32)).bfloat16()
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}
    ids = np.arange(20) * 7 % 512
    outs = []
    for s in (None, scaling):
        model = BitNetModel(dict(cfg, rope_scaling=s), use_gpu=True)
        model.load_state(state)
        assert np.array_equal(model._dev.rope.cpu().numpy(), rope_table(64, 128, 500000.0, s))
        outs.append(model.forward(ids)[0])
    assert np.isfinite(outs[1]).all() and not np.array_equal(outs[0], outs[1])
