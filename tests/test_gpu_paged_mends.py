"""The paged KV cache on the GPU, where calls are joined, captured or laid out in ways of their own; tolerances as in
test_gpu_paged.py unless a test derives its own."""
import math

import pytest
import torch

import test_gpu_paged as P
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def workspace(H, cache, table, weights):
    """Bytes that a call's pieces need: above 0 where it may cut a sequence."""
    from rotor.gpu_ternary import _paged_types, _paged_workspace_bytes

    Hkv, page, hd = cache.shape[2:]
    return _paged_workspace_bytes(_paged_types()[cache.dtype], Hkv, page, hd, *table.shape, H, weights)


# ---- weights -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", P.TYPES)
@pytest.mark.parametrize("slots", [200, 900, 4000])  # one piece; joined by the last workgroup; by a second launch
@pytest.mark.parametrize("bad", ["", "query", "key"])
def test_weights_of_holes(hip, dtype, slots, bad):
    """A hole's weights keep every bit: -0 stays -0, and a head whose query or key is NaN leaves its NaN at the slots it attends to."""
    cache, table, n = P.make([slots, slots - 7], 2, 64, 64, dtype)
    q = P.queries([0] * 2, 8, 64)
    if bad == "query":
        q[0, 0, 1, 3] = math.nan
    if bad == "key":
        cache[0, table[0, 0].long(), 0, 5, 9] = math.nan
    table[0, 1], table[1, 2] = -1, cache.shape[1]
    start = torch.full((2, 2, table.shape[1] * 64 + 4), -0.0)
    start[0, 0, 100] = 7.0
    w = start.cuda()
    hip.paged_attention(q.cuda(), cache.cuda(), table.cuda(), n.cuda(), weights=w)
    w = w.cpu()
    t = torch.arange(start.shape[2])
    for b in range(2):
        there = (t < n[b]) & (t // 64 != 1 + b)
        assert torch.equal(w[b, :, ~there].view(torch.int32), start[b, :, ~there].view(torch.int32)), b
        for h in range(2):
            nan = bad and b == 0 and h == 0
            assert w[b, h, there].isnan().all() if nan else (w[b, h, there] > 0).all()


def test_weights_over_a_wider_table(hip):
    """An eviction to more pages than there were: weights whose rows have the room go on, others are refused by the next step."""
    cache, table, n = P.make([90, 40], 2, 64, 16, "bf16", spare=22)
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))[:20].view(2, 10).int().cuda()
    k, rope = torch.randn(2, 1, 2, 64, device="cuda"), P.rope_angles(200, 64).cuda()
    for slots in (6 * 16, 10 * 16):
        w = torch.rand(2, 2, slots, device="cuda")
        c, pos = cache.cuda(), n.cuda()
        kept, lens, left = hip.paged_evict(c, table.cuda(), n.cuda(), w, 120, 5, free)
        assert lens.tolist() == [90, 40] and left.shape == w.shape and torch.equal(left[0, :, :90], w[0, :, :90])
        args = (P.queries([0] * 2, 8, 64).cuda(), k, k, c, free, lens, rope, pos)
        if slots < 160:
            with pytest.raises(ValueError, match="weights"):
                hip.paged_step(*args, weights=left)
        else:
            before = left.clone()
            hip.paged_step(*args, weights=left)
            assert (left[0, :, :91] > before[0, :, :91]).all() and (left[1, :, :41] > before[1, :, :41]).all()
            assert (left[0, :, 91:] == 0).all() and (left[1, :, 41:] == 0).all()


# ---- together with torch's graphs ----------------------------------------------------------


STEPS = {  # lens, H, Hkv, hd, page, dtype, weights, slots of the table beyond the lengths
    "last workgroup, weights in the launch": ([900], 20, 5, 128, 64, "bf16", True, 20),
    "last workgroup": ([900, 350, 0], 20, 5, 128, 64, "bf16", False, 20),
    "second launch, weights": ([4000, 30], 20, 5, 128, 64, "bf16", True, 20),
    "second launch": ([9000], 8, 2, 64, 128, "fp16", False, 20),
    "second launch, 1024 threads": ([1800, 3, 700], 14, 2, 64, 32, "fp32", True, 20),
    "last workgroup, tiles of heads": ([480, 300, 0], 40, 2, 64, 32, "bf16", False, 20),
    "second launch, tiles of heads": ([2900, 100], 50, 1, 128, 64, "fp16", True, 20),
    "more sequences than lanes": ([10 * b for b in range(70)], 4, 2, 64, 32, "bf16", True, 300),
}


@pytest.mark.parametrize("name", STEPS)
def test_replayed_steps_that_are_joined(hip, name):
    """Two captured steps that advance by themselves, in one workspace of the caller's that holds anything between the replays;
    every replay equal to the eager call on the same state, and that to the definition."""
    from rotor import _hip

    lens, H, Hkv, hd, page, dtype, weighted, extra = STEPS[name]
    cache, table, n = P.make(lens, Hkv, hd, page, dtype, extra=extra)
    B, t, need = len(lens), table.cuda(), workspace(H, cache, table, weighted)
    assert need > 0
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((B, 1, m, hd), generator=gen).cuda() for m in (H, Hkv, Hkv))
    rope = P.rope_angles(max(lens) + extra, hd).cuda()
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    class State:
        def __init__(self):
            self.cache, self.lens = cache.cuda(), n.cuda()
            self.w = torch.zeros((B, Hkv, t.shape[1] * page), device="cuda") if weighted else None
            self.out = torch.zeros_like(q)

        def call(self):
            c = self.cache
            pages = _hip.PAGES.pack(c.data_ptr(), c.stride(0), c.stride(1), t.data_ptr(), self.lens.data_ptr(), {"fp32": 0, "bf16": 1, "fp16": 2}[dtype],
                                    c.shape[1], Hkv, page, hd, B, t.shape[1])
            new = _hip.PAGED_NEW.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), rope.data_ptr(), self.lens.data_ptr(), 0, rope.shape[0], hd, 0, 1, H)
            hip._bind_stream()
            _hip.check(hip.lib.rt_paged_step(hip.ctx, pages, new, self.w.data_ptr() if weighted else None, t.shape[1] * page,
                                             self.out.data_ptr(), ws.data_ptr(), need))
            self.lens += 1

    a, b, e = State(), State(), State()
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                s.call()
    torch.cuda.current_stream().wait_stream(side)
    bits = torch.int32 if dtype == "fp32" else torch.int16
    for i, fill in enumerate([lambda: ws.fill_(255), lambda: ws.random_(0, 256), lambda: ws.zero_(), lambda: None, lambda: ws.fill_(1), lambda: None]):
        old = (e.w.cpu() if weighted else None, e.lens.cpu())
        e.call()
        for g in graphs:
            fill()
            g.replay()
        for s in (a, b):
            assert torch.equal(s.out, e.out) and torch.equal(s.lens, e.lens) and torch.equal(s.cache.view(bits), e.cache.view(bits)), i
            assert not weighted or torch.equal(s.w, e.w), i
        torch.cuda.synchronize()
        if i in (0, 5):  # (the queries as paged_append turns them)
            turned = hip.paged_append(q, k, v, e.cache.clone(), t, old[1].cuda(), rope, old[1].cuda())

            def once(w):
                if weighted:
                    w.copy_(e.w)
                return e.out

            P.check_attention(hip, e.cache.cpu(), table, e.lens.cpu(), turned.cpu(), weights=old[0], call=once)


def test_replayed_steps_whose_memory_is_used_again(hip):
    """Through the Python entry point: within a graph, the step's workspace is memory that other tensors of the graph have next."""
    cache, table, n = P.make([1500, 900], 5, 128, 64, "bf16", extra=10)
    need = workspace(20, cache, table, True)
    assert need > 0
    q, k = P.queries([0] * 2, 20, 128).cuda(), torch.randn(2, 1, 5, 128, device="cuda")
    rope, t = P.rope_angles(1600, 128).cuda(), table.cuda()

    def state():
        return [cache.cuda(), n.cuda(), torch.zeros(2, 5, t.shape[1] * 64, device="cuda")]

    def step(s, value):
        outs = [hip.paged_step(q, k, k, s[0], t, s[1], rope, s[1], weights=s[2])]
        torch.full((need,), value, dtype=torch.uint8, device="cuda")
        s[1] += 1
        outs.append(hip.paged_attention(q, s[0], t, s[1]))
        torch.full((need,), 255 - value, dtype=torch.uint8, device="cuda")
        return outs

    a, e = state(), state()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        got = step(a, 3)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(6):
        want = step(e, i)
        g.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a[2], e[2]), i
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", P.TYPES)
@pytest.mark.parametrize("lens,H,Hkv", [
    ([500, 300, 7], 20, 1), ([500] * 5 + [1], 40, 2), ([250, 100], 33, 1), ([130] * 30, 64, 2), ([6000, 0, 50], 130, 2), ([20000], 64, 1),
    ([700 + 9 * b for b in range(40)], 48, 1), ([300] * 66 + [5000], 34, 2)])
@pytest.mark.parametrize("weights", [False, True])
def test_tiles_of_heads_in_pieces(hip, dtype, lens, H, Hkv, weights):
    """Two to five tiles of heads a KV head, joined in both ways, in numbers of workgroups that 8 dies divide and that they do not."""
    cache, table, n = P.make(lens, Hkv, 64, 32, dtype, seed=H)
    start = torch.rand((len(lens), Hkv, table.shape[1] * 32), generator=torch.Generator().manual_seed(3)) if weights else None
    assert workspace(H, cache, table, weights) > 0
    check = P.check_attention(hip, cache, table, n, P.queries(lens, H, 64), weights=start)
    assert torch.equal(check, hip.paged_attention(P.queries(lens, H, 64).cuda(), cache.cuda(), table.cuda(), n.cuda(),
                                                  weights=start.cuda() if weights else None))


# ---- tokens without a place ----------------------------------------------------------------


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("held,heads", [(1500, 4), (1500, 16), (9000, 4)])
def test_step_without_a_place_that_is_joined(hip, weights, held, heads):
    """No page, no slot, no angle, over caches that are cut into pieces: nothing written, zeros, weights left, and the others as they
    would be."""
    page, hd = 64, 64
    cache, table, _ = P.make([held] * 6, 1, hd, page, "bf16", extra=page)
    cap = table.shape[1] * page
    assert workspace(heads, cache, table, weights) > 0
    table[1, held // page] = -1
    lens = torch.tensor([held, held, cap, -1, held, held], dtype=torch.int32)
    pos = torch.tensor([40, 40, 40, 40, 50, -1], dtype=torch.int32)
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((6, 1, n, hd), generator=gen) for n in (heads, 1, 1))
    rope = P.rope_angles(50, hd)
    start = torch.rand((6, 1, cap), generator=gen)
    c, w = cache.cuda(), start.cuda() if weights else None
    out = hip.paged_step(*(x.cuda() for x in (q, k, v)), c, table.cuda(), lens.cuda(), rope.cuda(), pos.cuda(), weights=w).cpu()
    assert (out[1:] == 0).all()
    if weights:
        assert torch.equal(w[1:].cpu(), start[1:])
    changed = (c.cpu().float().nan_to_num(7.0) != cache.float().nan_to_num(7.0)).any(-1).nonzero()
    assert {(int(p), int(r)) for _, p, _, r in changed} == {(int(table[0, held // page]), held % page)}
    turned, _ = PO.append(q[:1], k[:1], v[:1], cache, table[:1], lens[:1], rope, pos[:1])
    n = torch.tensor([held + 1], dtype=torch.int32)

    def first(wd):
        if weights:
            wd.copy_(w[:1])
        return out[:1]

    P.check_attention(hip, c.cpu(), table[:1], n, turned.float(), weights=start[:1] if weights else None, call=first)


# ---- layouts -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", P.TYPES)
def test_layers_of_one_tensor(hip, dtype):
    """Append, step and eviction on a layer whose pages hold keys next to values, between other layers: as on a cache of its own, and
    nothing else is touched."""
    B, H, Hkv, hd, page, keep = 2, 8, 2, 64, 32, 40
    cache, table, n = P.make([90, 40], Hkv, hd, page, dtype, extra=12, spare=6)
    free = torch.tensor(sorted(set(range(cache.shape[1])) - set(table.flatten().tolist())))[:4].view(2, 2).int().cuda()
    gen = torch.Generator().manual_seed(6)
    bits = torch.int32 if dtype == "fp32" else torch.int16
    layers = torch.randn((cache.shape[1], 3, 2, *cache.shape[2:]), generator=gen).to(cache.dtype).cuda()
    layers[:, 1] = cache.cuda().transpose(0, 1)
    others = layers[:, ::2].clone()
    near, apart = layers[:, 1].transpose(0, 1), cache.cuda()
    assert not near.is_contiguous()
    new = lambda M: [torch.randn((B, M, m, hd), generator=gen).cuda() for m in (H, Hkv, Hkv)]  # noqa: E731
    rope, t, lens = P.rope_angles(200, 32).cuda(), table.cuda(), n.cuda()
    prompt, one, w = new(9), new(1), torch.rand((B, Hkv, table.shape[1] * page), generator=gen).cuda()
    runs = []
    for c in (near, apart):
        weights = w.clone()
        outs = [hip.paged_append(*prompt, c, t, lens, rope, lens), c.clone()]
        outs += [hip.paged_step(*one, c, t, lens + 9, rope, lens + 9, weights=weights), c.clone(), weights]
        outs += [*hip.paged_evict(c, t, lens + 10, weights, keep, 7, free), c.clone()]
        runs.append(outs)
    for x, y in zip(*runs):
        assert torch.equal(x.contiguous().view(bits if x.dtype == cache.dtype else torch.int32),
                           y.contiguous().view(bits if x.dtype == cache.dtype else torch.int32))
    assert torch.equal(layers[:, ::2].view(bits), others.view(bits))


# ---- accuracy ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", P.TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_every_bit_of_queries_and_weights(hip, dtype, hd):
    """Two slots, keys e_d and 0, values 1 and 0: the output is 1 / (1 + exp(-x / sqrt(hd))) for a query x e_d whose 24 bits all count.
    With s = x log2(e) / sqrt(hd): products and their sums are exact; the scale's constant, root and quotient and the product with it are
    off by 4 u |s|, which is no more than 4 ln 2 u |s| of a weight; exp2 by an ulp (2 u), sum, reciprocal and product by u each, and
    the splits of the weights by nothing: (4 |s| + 8) u of the output.  Queries, or weights, of two bf16 are off by up to 2^-15 of
    themselves, 512 u.  Another dimension of the query, where the keys are 0, is 2^20 times as large and must not cost it bits."""
    H, gen = 64, torch.Generator().manual_seed(hd)
    x = (torch.rand(H, generator=gen) * 8 - 4) * math.sqrt(hd) / math.log2(math.e)
    table, n = torch.tensor([[1]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    for d, big in ((5, None), (hd - 1, 3), (33, 60)):
        cache = torch.full((2, 3, 1, 16, hd), math.nan, dtype=P.TYPES[dtype])
        cache[:, 1, :, :2] = 0
        cache[0, 1, 0, 0, d], cache[1, 1, 0, 0] = 1, 1
        q = torch.zeros(1, 1, H, hd)
        q[0, 0, :, d] = x
        if big is not None:
            q[..., big] = x.abs().max() * 2.0 ** 20
        s = x.double() * math.log2(math.e) / math.sqrt(hd)
        want = (1 / (1 + torch.exp2(-s)))[None, None, :, None]
        got = hip.paged_attention(q.cuda(), cache.cuda(), table.cuda(), n.cuda()).cpu().double()
        bound = (4 * s.abs() + 8)[None, None, :, None] * U * want
        assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


# ---- a model's angles ------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 4])
def test_model_with_angles_scaled_by_two(hip, bits):
    """The first layer's keys at position 2 p under linear scaling by 2 are those of the same token at p without it, bit for bit: in a
    prompt and in single steps."""
    import numpy as np

    import test_gpu_model as T
    from oracle import rotor_oracle as O

    params = O.make_bitnet_params(77, T.SMALL, 96)
    ids = np.random.default_rng(2).integers(0, T.SMALL["vocab_size"], 21).astype(np.int32)
    twice = np.repeat(ids, 2)
    keys = []
    for scaling, seq in ((None, ids), ({"rope_type": "linear", "factor": 2.0}, twice)):
        model = T._device_model(hip, params, dict(T.SMALL, kv_cache_bits=bits, rope_scaling=scaling), 96)
        first = len(seq) // 3 * 2 // 2 * 2
        _, cache = model.forward(seq[:first], use_cache=True)
        for token in seq[first:]:
            _, cache = model.forward(np.array([token], np.int32), past_kv_cache=cache, use_cache=True)
        keys.append(np.asarray(cache[0]["k"]))
    assert keys[0].shape[2] == 21 and keys[1].shape[2] == 42
    assert np.array_equal(keys[0], keys[1][:, :, ::2]) and not np.array_equal(keys[0], keys[1][:, :, :21])
