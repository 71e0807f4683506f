"""A paged KV cache, the decoding over it and the eviction from it: what is measured of them.

Kinds of case (the field "kind"):
  append  RoPE of queries and keys, keys and values into the pages: the rotated queries and the cache
  step    one new token a sequence: append, and attention over all it then holds: the attention's
          output, the cache, and the accumulated weights where the case keeps them
  attend  attention of one token a sequence over what the cache holds (and the accumulated weights)
  evict   what is kept of a cache that is to shrink, by accumulated weight, copied to other pages: the
          slots kept, how many, the cache, and their weights

The cache of a layer is [2 (K, V), pages, Hkv, page, hd].  Slot t of sequence b is row t % page of page
table[b, t / page]; lens[b] slots are held, and `pos` is the position that the next token's angles
have, `ahead` past lens (what was evicted counts there).  Memory that nothing was written to is NaN, and
a table's entries past what its sequence needs are -1.  The sequences of a batch are of lengths spread from `lo` to
`hi`; sizes are those of the benchmark's model (20 query and 5 KV heads of 128) and generic ones.
"""
import math
import sys

import torch

own = False

THETA = 500000.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    model = dict(H=20, Hkv=5, hd=128, dtype="bf16", page=64)
    half = dict(rotary=128, interleaved=False, scaled=False, ahead=0, ragged=False)
    return [
        # one token of a chat enters the cache (the smallest call)
        dict(name="append_1", kind="append", B=1, M=1, lo=1537, hi=1537, **model, **half),
        # a step of 64 sequences whose caches were cut, angles for half of each head, small heads and pages
        dict(name="append_64", kind="append", B=64, M=1, H=16, Hkv=8, hd=64, dtype="fp16", page=16, lo=3, hi=999, rotary=32,
             interleaved=True, scaled=False, ahead=4000, ragged=False),
        # prompts of different lengths, each behind what it has, angles scaled for a longer context
        dict(name="append_8x2048", kind="append", B=8, M=2048, lo=0, hi=6144, **model, **dict(half, scaled=True, ragged=True)),
        # one token of a chat through a layer's attention
        dict(name="step_1537", kind="step", B=1, weights=False, lo=1537, hi=1537, **model, **half),
        # a step of a busy server that keeps the weights for a later eviction
        dict(name="step_20_weights", kind="step", B=20, weights=True, lo=50, hi=6000, **dict(model, H=32, Hkv=8), **half),
        # a step of 32 sequences of ragged lengths
        dict(name="attend_32", kind="attend", B=32, weights=False, lo=100, hi=4095, **model),
        # one token after a very long document
        dict(name="attend_131072", kind="attend", B=1, weights=False, lo=131071, hi=131071, **model),
        # heads that share nothing, small, with small pages
        dict(name="attend_8_mha", kind="attend", B=8, weights=False, H=12, Hkv=12, hd=64, dtype="fp16", page=16, lo=5, hi=776),
        # a cache in fp32, seven query heads to a KV head, one sequence that has nothing yet
        dict(name="attend_6_fp32_weights", kind="attend", B=6, weights=True, H=14, Hkv=2, hd=64, dtype="fp32", page=32, lo=0, hi=3001),
        # a chat's cache halved
        dict(name="evict_2048", kind="evict", B=1, keep=1024, recent=256, lo=2048, hi=2048, **model),
        # a server's sequences cut to a budget that some have not reached
        dict(name="evict_16", kind="evict", B=16, keep=4096, recent=512, H=16, Hkv=8, hd=64, dtype="fp16", page=32, lo=1000, hi=8191),
        # two very long documents cut to a quarter
        dict(name="evict_2x131072", kind="evict", B=2, keep=32768, recent=1000, lo=100000, hi=131072, **model),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    kind = rng.choice(["append", "step", "attend", "attend", "evict"])
    limit = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        Hkv, hd, B = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128]), _log(rng, 1, 64)
        case = dict(kind=kind, B=B, H=Hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), Hkv=Hkv, hd=hd,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), page=rng.choice([16, 32, 64, 128, 256]))
        most = _log(rng, 16, 131072)
        case["lo"], case["hi"] = sorted(rng.randint(0, most) for _ in range(2))
        if kind in ("append", "step"):
            case.update(rotary=rng.choice([hd, hd, hd // 2, hd // 4, 24]), interleaved=rng.random() < 0.4, scaled=rng.random() < 0.3,
                        ahead=rng.choice([0, 0, _log(rng, 1, 20000)]), ragged=False)
        if kind == "append":
            case.update(M=_log(rng, 1, 2048), ragged=rng.random() < 0.4)
        elif kind == "evict":
            case["keep"] = rng.randint(1, max(1, case["hi"]))
            case["recent"] = rng.randint(0, case["keep"])
        else:
            case["weights"] = rng.random() < 0.4
        if _cost(case) <= limit and B * Hkv * case["hi"] * hd <= 1 << 27:
            return case


def _lens(case):
    """Each sequence's slots: the first hi, the last lo, the others between by the golden ratio."""
    lo, hi, B = case["lo"], case["hi"], case["B"]
    lens = [hi - int((b * 0.6180339887498949) % 1.0 * (hi - lo + 1)) for b in range(B)]
    return lens[:-1] + [lo] if B > 1 else lens


def _counts(case):
    """The new tokens of each sequence: M, or for some fewer."""
    if case["kind"] != "append":
        return [1] * case["B"]
    M = case["M"]
    return [M - int((b * 0.6180339887498949) % 1.0 * (M // 2 + 1)) if case["ragged"] else M for b in range(case["B"])]


def _need(case):
    """Slots that each sequence has pages for."""
    if case["kind"] in ("append", "step"):
        return [n + c for n, c in zip(_lens(case), _counts(case))]
    return _lens(case)


def _kept(case):
    return [min(n, case["keep"]) for n in _lens(case)]


def work(case):
    B, H, Hkv, hd, lens = case["B"], case["H"], case["Hkv"], case["hd"], _lens(case)
    e = 4 if case["dtype"] == "fp32" else 2
    token = 2 * Hkv * hd * e  # a slot's key and value
    if case["kind"] == "evict":
        kept, slots = sum(_kept(case)), -(-max(max(lens), 1) // case["page"]) * case["page"]
        return {"bytes": 4 * Hkv * (sum(lens) + B * case["keep"] + B * slots) + 2 * token * kept, "flops": 4 * Hkv * sum(lens)}
    new = sum(_counts(case))
    into = new * (4 * (H + 2 * Hkv) * hd + token) + 4 * case.get("rotary", 0) * new  # q, k, v, the rows written, the angles
    turn = 3 * new * (H + Hkv) * case.get("rotary", 0)
    if case["kind"] == "append":
        return {"bytes": into + 4 * B * case["M"] * H * hd, "flops": turn}
    flops, out = 4 * H * hd * sum(lens), 4 * B * H * hd
    read = sum(lens) * (token + 8 * Hkv * case["weights"]) + out
    if case["kind"] == "attend":
        return {"bytes": read + out, "flops": flops}
    return {"bytes": read + into, "flops": flops + turn}


# ---- inputs ------------------------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _heads(gen, *shape):
    """Queries or keys [.., heads, hd]: one channel in sixteen is four times as wide, and channels have a mean."""
    wide = torch.where(torch.rand(shape[-2:], generator=gen, device="cuda") < 1 / 16, 4.0, 1.0)
    return _normal(gen, *shape) * wide + 0.5 * _normal(gen, *shape[-2:])


def _angles(rows, rotary, scaled):
    """(cos, sin) of position * frequency: fp32 [rows, rotary / 2, 2], computed in 64 bits.  Scaled: frequencies of fewer
    than one turn in the original context go four times as slowly, those of more than 32 turns stay, those between are
    mixed, and the vectors grow by 0.1 ln 4 (YaRN)."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    f, grow = THETA ** (-2.0 * i / rotary), 1.0
    if scaled:
        at = [rotary * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(THETA)) for turns in (32, 1)]
        first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        slow = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        f, grow = f / 4 * slow + f * (1 - slow), 0.1 * math.log(4) + 1
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * f
    return (torch.stack([a.cos(), a.sin()], -1) * grow).float()


def _tables(gen, needs, page, pages):
    """Tables int32 [B, P] for each list of slots in `needs`, over different pages of a shuffled pool."""
    order, at, out = torch.randperm(pages, generator=gen, device="cuda").int(), 0, []
    for need in needs:
        n = torch.tensor([-(-x // page) for x in need], device="cuda")
        first = at + n.cumsum(0) - n
        j = torch.arange(max(1, int(n.max())), device="cuda")
        out.append(torch.where(j < n[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], -1))
        at += int(n.sum())
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hkv, hd, page = (case[k] for k in ("B", "H", "Hkv", "hd", "page"))
    needs = [_need(case)] + ([[case["keep"]] * B] if case["kind"] == "evict" else [])
    pages = sum(-(-x // page) for need in needs for x in need) + 3
    cache = torch.full((2, pages, Hkv, page, hd), math.nan, dtype=TYPES[case["dtype"]], device="cuda")
    tables = _tables(gen, needs, page, pages)
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    b, t = (torch.arange(tables[0].shape[1] * page, device="cuda") < lens[:, None]).nonzero(as_tuple=True)  # the slots held
    at = tables[0][b, t // page].long()
    cache[0, at, :, t % page] = _heads(gen, len(b), Hkv, hd).to(cache.dtype)
    cache[1, at, :, t % page] = _normal(gen, len(b), Hkv, hd).to(cache.dtype)
    st = dict(case, cache=cache, table=tables[0], lens=lens)
    if case["kind"] == "evict":
        st["new_table"] = tables[1]
    else:
        M = case.get("M", 1)
        st["q"] = _heads(gen, B, M, H, hd)
    if case["kind"] in ("append", "step"):
        st.update(k=_heads(gen, B, M, Hkv, hd), v=_normal(gen, B, M, Hkv, hd), pos=lens + case["ahead"],
                  rope=_angles(case["hi"] + case["ahead"] + M, case["rotary"], case["scaled"]))
        st["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    if case["kind"] == "evict" or case.get("weights"):
        w = torch.exp(2 * _normal(gen, B, Hkv, tables[0].shape[1] * page)) / 64
        st["weights"] = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.1, 0.0, w)  # (ties)
    else:
        st["weights"] = None
    return st


# ---- the plain forms ---------------------------------------------------------------------


def rotate(x, cs, rows, interleaved):
    """RoPE of x [B, M, heads, hd] at positions rows [B, M]: in 64 bits, rounded once."""
    n = cs.shape[1]
    c, s = cs[rows].double()[:, :, None].unbind(-1)
    y = x[..., :2 * n].double()
    a, b = (y[..., ::2], y[..., 1::2]) if interleaved else (y[..., :n], y[..., n:])
    turned = torch.stack([a * c - b * s, b * c + a * s], -1 if interleaved else -2).flatten(-2)
    return torch.cat([turned.float(), x[..., 2 * n:]], -1)


def _put(st):
    """The new rows into the cache; the rotated queries."""
    m = torch.arange(st["q"].shape[1], device="cuda")
    counts = st["counts"][:, None] if st["counts"] is not None else len(m)
    there = m < counts
    rows = (st["pos"][:, None] + m).long().clamp(max=len(st["rope"]) - 1)
    q, k = (rotate(x, st["rope"], rows, st["interleaved"]) for x in (st["q"], st["k"]))
    b, m = there.expand(st["B"], -1).nonzero(as_tuple=True)
    slot = st["lens"][b] + m
    at = st["table"][b, slot // st["page"]].long()
    st["cache"][0, at, :, slot % st["page"]] = k[b, m].to(st["cache"].dtype)
    st["cache"][1, at, :, slot % st["page"]] = st["v"][b, m].to(st["cache"].dtype)
    return torch.where(there[..., None, None], q, 0.0) if st["counts"] is not None else q


def _attend(st, q, lens):
    B, H, Hkv, hd = q.shape[0], st["H"], st["Hkv"], st["hd"]
    K, V = (x[st["table"].long().clamp(min=0)].transpose(1, 2).reshape(B, Hkv, -1, hd).float() for x in st["cache"])
    hidden = (torch.arange(K.shape[2], device="cuda") >= lens[:, None])[:, None, :, None]
    K, V = K.masked_fill(hidden, 0.0), V.masked_fill(hidden, 0.0)
    s = (q.view(B, Hkv, H // Hkv, hd) @ K.transpose(2, 3) / math.sqrt(hd)).masked_fill(hidden.transpose(2, 3), -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    if st["weights"] is not None:
        st["weights"] += p.sum(2)
    return (p @ V).view(B, 1, H, hd)


def _evict(st):
    w, lens, page, keep = st["weights"], st["lens"], st["page"], st["keep"]
    B, Hkv, slots = w.shape
    t, n = torch.arange(slots, device="cuda"), lens[:, None, None]
    order = torch.where(t < n, w, -1.0).masked_fill((t < n) & (t >= n - st["recent"]), math.inf)
    chosen = order.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values  # in order of their slots
    chosen = torch.nn.functional.pad(chosen, (0, keep - chosen.shape[-1]), value=slots)
    new_lens = lens.clamp(max=keep)
    there = torch.arange(keep, device="cuda") < new_lens[:, None, None]
    kept = torch.where(there, chosen, -1)
    b, h, i = there.expand(B, Hkv, keep).nonzero(as_tuple=True)
    t = kept[b, h, i]
    st["cache"][:, st["new_table"][b, i // page].long(), h, i % page] = st["cache"][:, st["table"][b, t // page].long(), h, t % page]
    weights = torch.zeros_like(w)
    weights[b, h, i] = w[b, h, t]
    return kept.int(), new_lens, st["cache"], weights


def run(st):
    if own:
        return _own(st, _backend())
    if st["kind"] == "evict":
        return _evict(st)
    if st["kind"] == "append":
        return _put(st), st["cache"]
    if st["kind"] == "step":
        out = (_attend(st, _put(st), st["lens"] + 1), st["cache"])
    else:
        out = (_attend(st, st["q"], st["lens"]),)
    return out if st["weights"] is None else (*out, st["weights"])


def _own(st, hip):
    cache, table, lens = st["cache"], st["table"], st["lens"]
    if st["kind"] == "evict":
        kept, new_lens, weights = hip.paged_evict(cache, table, lens, st["weights"], st["keep"], st["recent"], st["new_table"])
        return kept, new_lens, cache, weights
    if st["kind"] == "append":
        return hip.paged_append(st["q"], st["k"], st["v"], cache, table, lens, st["rope"], st["pos"], counts=st["counts"],
                                interleaved=st["interleaved"]), cache
    if st["kind"] == "step":
        out = (hip.paged_step(st["q"], st["k"], st["v"], cache, table, lens, st["rope"], st["pos"], interleaved=st["interleaved"],
                              weights=st["weights"]), cache)
    else:
        out = (hip.paged_attention(st["q"], cache, table, lens, weights=st["weights"]),)
    return out if st["weights"] is None else (*out, st["weights"])


def _backend():
    if "rotor-rag_amd" not in sys.path:
        sys.path.insert(0, "rotor-rag_amd")
    from rotor.gpu_layers import get_gpu, last_error

    hip = get_gpu()
    if hip is None:
        raise RuntimeError(last_error())
    return hip


# ---- the definition, in 64 bits ----------------------------------------------------------


def _turned(x, angle, interleaved):
    """x float64 [M, heads, hd], angle [M, rotary / 2, 2]: the pairs as complex numbers, times the angle's."""
    n = angle.shape[1]
    pairs = torch.empty((*x.shape[:2], n, 2), dtype=torch.float64, device="cuda")
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    pairs[..., 0], pairs[..., 1] = x[..., first], x[..., second]
    z = torch.view_as_complex(pairs) * torch.view_as_complex(angle.contiguous())[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _slots(st, b, first, last):
    """(page, row) of slots [first, last) of sequence b."""
    t = torch.arange(first, last, device="cuda")
    return st["table"][b].long()[t // st["page"]], t % st["page"]


def exact(case, seed):
    st = prepare(case, seed)
    cache = st["cache"].double()
    lens, counts, G = _lens(case), _counts(case), case["H"] // case["Hkv"]
    weights = st["weights"].double() if st["weights"] is not None else None
    if case["kind"] == "evict":
        kept = torch.full((case["B"], case["Hkv"], case["keep"]), -1, dtype=torch.int32, device="cuda")
        left = torch.zeros_like(weights)
        for b, n in enumerate(lens):
            old = max(0, n - case["recent"])  # slots that are judged
            extra = min(case["keep"], n) - (n - old)
            for h in range(case["Hkv"]):
                best = torch.argsort(-weights[b, h, :old], stable=True)[:extra]
                t = torch.cat([best.sort().values, torch.arange(old, n, device="cuda")])
                i = torch.arange(len(t), device="cuda")
                kept[b, h, :len(t)] = t.int()
                left[b, h, :len(t)] = weights[b, h, t]
                to, frm = st["new_table"][b].long()[i // case["page"]], st["table"][b].long()[t // case["page"]]
                cache[:, to, h, i % case["page"]] = cache[:, frm, h, t % case["page"]]
        return kept, torch.tensor(_kept(case), dtype=torch.int32, device="cuda"), cache, left
    q = st["q"].double()
    if case["kind"] != "attend":
        for b, (n, c) in enumerate(zip(lens, counts)):
            angle = st["rope"][n + case["ahead"]:n + case["ahead"] + c].double()
            q[b, :c], q[b, c:] = _turned(q[b, :c], angle, case["interleaved"]), 0.0
            page, row = _slots(st, b, n, n + c)
            cache[0, page, :, row] = _turned(st["k"][b, :c].double(), angle, case["interleaved"]).to(st["cache"].dtype).double()
            cache[1, page, :, row] = st["v"][b, :c].to(st["cache"].dtype).double()
    if case["kind"] == "append":
        return q, cache
    out = torch.zeros_like(q)
    for b, n in enumerate(lens):
        n += case["kind"] == "step"
        page, row = _slots(st, b, 0, n)
        for h in range(case["Hkv"] if n else 0):
            K, V = cache[0, page, h, row], cache[1, page, h, row]
            p = torch.softmax(q[b, 0, h * G:(h + 1) * G] @ K.T.contiguous() / case["hd"] ** 0.5, -1)
            out[b, 0, h * G:(h + 1) * G] = p @ V
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    outs = [out] + ([cache] if case["kind"] == "step" else [])
    return tuple(outs if weights is None else outs + [weights])
