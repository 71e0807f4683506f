"""The 4-bit KV cache and the attention that reads it: what is measured of them.

Kinds of case (the field "kind"):
  write      RoPE of queries and keys, keys and values into the cache in 4 bits, and the new
             positions read back: the rotated queries and the keys and values as later steps see them
  read       every cached position of a layer back as fp32 keys and values
  attention  causal GQA attention of the M newest tokens of each sequence over its cached positions
             (M = 1: a decode step; more: a prompt, or one chunk of it)

The sequences of a batch stand at positions of their own, spread from `lo` to `hi`; sizes are those
of the benchmark's model (20 query and 5 KV heads of 128) and generic ones.

The cache of a layer is uint8 [B, Hkv, blocks of 64 positions, block bytes].  A group is 64
consecutive dimensions of one head at one position, held as codes c = 0..15 and two bf16 numbers: the
middle z and the half step h, value = z + h (2 c - 15).  A block holds, in little-endian dwords,
  K codes   [64 positions][4 h][hd/64 g][2 e]: dimensions 64 g + 16 h + 8 e + (0..7)
  V codes   [hd/32 u][16 d][4 = 2 s + l][2 v][2 w]: dimension 32 u + 16 v + d, positions
            32 w + 16 s + 4 l + (0, 1, 2, 3, 8, 9, 10, 11)
  K scales  [hd/64][64 positions]: z << 16 | h;   V scales the same
and element e of a dword's eight lies in its nibble e / 2 + 4 (e % 2).
"""
import math
import sys

import torch

own = False

THETA = 500000.0
H, HKV, HD = 20, 5, 128  # the benchmark model's heads


def listed():
    model = dict(H=H, Hkv=HKV, hd=HD)
    return [
        # one token's keys and values enter the cache of a chat (the smallest call)
        dict(name="write_1", kind="write", B=1, M=1, Lmax=2048, lo=1537, hi=1537, **model),
        # a step of 64 sequences, small heads, lengths all over
        dict(name="write_batch_64", kind="write", B=64, M=1, H=16, Hkv=8, hd=64, Lmax=1000, lo=3, hi=999),
        # long prompts of several sequences, each behind what it has already
        dict(name="write_8x2048", kind="write", B=8, M=2048, Lmax=8192, lo=0, hi=6144, **model),
        # a layer's cache read back, as a caller who looks at it does
        dict(name="read_1538", kind="read", B=1, M=1538, Hkv=HKV, hd=HD, Lmax=2048),
        # long sequences read back whole, to be moved or stored elsewhere
        dict(name="read_4x32768", kind="read", B=4, M=32768, Hkv=HKV, hd=HD, Lmax=32768),
        # one token of a chat: the smallest attention
        dict(name="decode_1537", kind="attention", B=1, M=1, Lmax=2048, lo=1537, hi=1537, **model),
        # a decode step of 32 sequences of ragged lengths
        dict(name="decode_32", kind="attention", B=32, M=1, Lmax=4096, lo=100, hi=4095, **model),
        # one token after a very long document
        dict(name="decode_131072", kind="attention", B=1, M=1, Lmax=131072, lo=131071, hi=131071, **model),
        # heads that share nothing, small, an odd length
        dict(name="decode_8_mha", kind="attention", B=8, M=1, H=12, Hkv=12, hd=64, Lmax=777, lo=5, hi=776),
        # the benchmark's prompt, into an empty cache
        dict(name="prefill_512", kind="attention", B=1, M=512, Lmax=640, lo=0, hi=0, **model),
        # the last chunk of a long prompt
        dict(name="prefill_2048_of_8192", kind="attention", B=1, M=2048, Lmax=8192, lo=6144, hi=6144, **model),
        # three ragged chunks, seven query heads to a KV head
        dict(name="prefill_3x77", kind="attention", B=3, M=77, H=14, Hkv=2, hd=64, Lmax=1111, lo=0, hi=1001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    shape = rng.choice(["write", "read", "decode", "decode", "prefill"])
    limit = max(_cost(c) for c in listed() if c["kind"] == ("attention" if shape in ("decode", "prefill") else shape)
                and (shape not in ("decode", "prefill") or (c["M"] == 1) == (shape == "decode")))
    while True:
        Hkv = rng.choice([1, 2, 3, 4, 5, 8])
        heads = dict(H=Hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), Hkv=Hkv, hd=rng.choice([64, 128]))
        B = _log(rng, 1, 64)
        Lmax = _log(rng, 64, 131072)
        if shape == "read":
            del heads["H"]
            case = dict(kind="read", B=B, M=_log(rng, 1, Lmax), Lmax=Lmax, **heads)
        else:
            M = 1 if shape == "decode" else min(Lmax, _log(rng, 1 if shape == "write" else 2, 2048))
            ends = sorted(rng.randint(0, Lmax - M) for _ in range(2))
            case = dict(kind="write" if shape == "write" else "attention", B=B, M=M, Lmax=Lmax, lo=ends[0], hi=ends[1],
                        **heads)
        if _cost(case) <= limit and B * Hkv * Lmax * case["hd"] <= 1 << 27:
            return case


def _positions(case):
    """Each sequence's position, spread over [lo, hi] by the golden ratio (the first at hi)."""
    if case["kind"] == "read":
        return [0] * case["B"]
    lo, hi = case["lo"], case["hi"]
    return [hi - int((b * 0.6180339887498949) % 1.0 * (hi - lo + 1)) for b in range(case["B"])]


def work(case):
    B, M, Hkv, hd = case["B"], case["M"], case["Hkv"], case["hd"]
    token = 2 * Hkv * (hd // 2 + hd // 16)  # a position in the cache: codes and scales of K and V
    if case["kind"] == "read":
        return {"bytes": B * M * (token + 8 * Hkv * hd), "flops": 4 * B * M * Hkv * hd}
    H_, pos = case["H"], _positions(case)
    if case["kind"] == "write":
        angles = len({p + m for p in set(pos) for m in range(M)})
        moved = 4 * (2 * H_ + 2 * Hkv) * hd + 2 * token + 8 * Hkv * hd  # q in and out, k, v, cache out and in, values
        return {"bytes": B * M * moved + 4 * hd * angles, "flops": B * M * hd * (3 * (H_ + Hkv) + 2 * Hkv * 10)}
    pairs = sum(M * p + M * (M + 1) // 2 for p in pos)
    return {"bytes": sum(p + M for p in pos) * token + 8 * B * M * H_ * hd, "flops": 4 * H_ * hd * pairs}


# ---- inputs ------------------------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _heads(gen, B, L, n, hd):
    """Queries or keys: one channel in sixteen is four times as wide, and channels have a mean."""
    wide = torch.where(torch.rand((n, hd), generator=gen, device="cuda") < 1 / 16, 4.0, 1.0)
    return _normal(gen, B, L, n, hd) * wide + 0.5 * _normal(gen, n, hd)


def _angles(Lmax, hd):
    """(cos, sin) of position * theta^(-2 i / hd): fp32 [Lmax, hd / 2, 2], computed in 64 bits."""
    i = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(Lmax, dtype=torch.float64, device="cuda")[:, None] * THETA ** (-2.0 * i / hd)
    return torch.stack([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, M, Hkv, hd, Lmax = (case[k] for k in ("B", "M", "Hkv", "hd", "Lmax"))
    blocks = -(-Lmax // 64)
    st = dict(case, pos=torch.tensor(_positions(case), dtype=torch.int32, device="cuda"))
    if case["kind"] == "write":
        st.update(q=_heads(gen, B, M, case["H"], hd), k=_heads(gen, B, M, Hkv, hd), v=_normal(gen, B, M, Hkv, hd),
                  rope=_angles(Lmax, hd))
        st["cache"] = torch.randint(0, 256, (B, Hkv, blocks, 72 * hd), generator=gen, device="cuda", dtype=torch.uint8)
        return st
    st["cache"] = pack(_heads(gen, B, blocks * 64, Hkv, hd).transpose(1, 2), _normal(gen, B, Hkv, blocks * 64, hd))
    if case["kind"] == "attention":
        st["q"] = _heads(gen, B, M, case["H"], hd)
    return st


# ---- the plain forms ---------------------------------------------------------------------


def rotate(x, cs, rows):
    """RoPE (rotate half) of x [B, M, heads, hd] at positions rows [B, M]: in 64 bits, rounded once."""
    half = x.shape[-1] // 2
    c, s = cs[rows].double()[:, :, None].unbind(-1)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1).float()


def quantise(x):
    """x fp32 [..., hd] -> codes int32 [..., hd], z and h as fp32 [..., hd / 64] (in 64 bits: codes
    next to a border are decided as they are)."""
    g = x.double().unflatten(-1, (-1, 64))
    lo, hi = 0.5 * g.amin(-1), 0.5 * g.amax(-1)
    z, h = (hi + lo).float().bfloat16().float(), ((hi - lo) / 15).float().bfloat16().float()
    lost = ~(torch.isfinite(g).all(-1) & torch.isfinite(z) & torch.isfinite(h))
    z, h = torch.where(lost, math.nan, z), torch.where(lost, 0.0, h)
    t = torch.where((h == 0)[..., None], 0.0, (g - z[..., None]) / h[..., None])
    return torch.clamp(torch.round((t + 15) / 2), 0, 15).to(torch.int32).flatten(-2), z, h


def scale_bits(z, h):
    """z << 16 | h, the bf16 bits, as int32."""
    return z.contiguous().view(torch.int32) | (h.contiguous().view(torch.int32) >> 16)


def _nibbles(c):
    """Codes [..., 8] -> int32 [...]: element e in nibble e / 2 + 4 (e % 2)."""
    at = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=c.device, dtype=torch.int32)
    return (c << at).sum(-1, dtype=torch.int32)


def pack(k, v):
    """Keys and values fp32 [B, Hkv, L, hd] (L a multiple of 64) -> the cache's bytes."""
    B, Hkv, L, hd = k.shape
    (ck, zk, hk), (cv, zv, hv) = quantise(k), quantise(v)
    kc = _nibbles(ck.view(B, Hkv, L // 64, 64, hd // 64, 4, 2, 8).transpose(4, 5))
    # positions 64 = (w, s, x, l, r), dimensions hd = (u, v, d): [u, d, s, l, v, w, (x, r)]
    vc = cv.view(B, Hkv, L // 64, 2, 2, 2, 2, 4, hd // 32, 2, 16).permute(0, 1, 2, 8, 10, 4, 6, 9, 3, 5, 7)
    vc = _nibbles(vc.reshape(*vc.shape[:-2], 8))
    ks, vs = (scale_bits(z, h).view(B, Hkv, L // 64, 64, hd // 64).transpose(3, 4) for z, h in ((zk, hk), (zv, hv)))
    return torch.cat([x.reshape(B, Hkv, L // 64, -1) for x in (kc, vc, ks, vs)], -1).view(torch.uint8)


def unpack(cache):
    """The cache's bytes -> keys and values fp32 [B, Hkv, L, hd]."""
    B, Hkv, n, size = cache.shape
    hd = size // 72
    kc, vc, ks, vs = cache.view(torch.int32).split([8 * hd, 8 * hd, hd, hd], -1)
    at = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=cache.device, dtype=torch.int32)
    kc = ((kc[..., None] >> at) & 15).view(B, Hkv, n, 64, 4, hd // 64, 2, 8).transpose(4, 5)
    vc = ((vc[..., None] >> at) & 15).view(B, Hkv, n, hd // 32, 16, 2, 2, 2, 2, 2, 4)
    vc = vc.permute(0, 1, 2, 8, 5, 9, 6, 10, 3, 7, 4)

    def values(c, scale):
        scale = scale.reshape(B, Hkv, n, hd // 64, 64).transpose(3, 4).reshape(B, Hkv, n * 64, hd // 64, 1)
        z, h = (scale & -65536).view(torch.float32), (scale << 16).view(torch.float32)
        return (z + h * (2 * c.reshape(B, Hkv, n * 64, hd // 64, 64) - 15)).flatten(-2)

    return values(kc, ks), values(vc, vs)


def _places(rows, hd, heads, blocks):
    """Where positions rows [B, M] lie in the cache as dwords: for K and for V the dword [B, M, heads, hd]
    and the shift in it of every element's code, and the dword [B, M, heads, hd / 64] of its scales."""
    dev = rows.device
    i, g = torch.arange(hd, device=dev), torch.arange(hd // 64, device=dev)
    b, n = torch.arange(rows.shape[0], device=dev)[:, None, None], torch.arange(heads, device=dev)
    base = (((b * heads + n) * blocks + (rows // 64)[:, :, None]) * (18 * hd))[..., None]
    p = (rows % 64)[:, :, None, None]
    shift = lambda e: 4 * (e // 2 + 4 * (e % 2))  # noqa: E731
    k_at = base + p * (hd // 8) + (i // 16 % 4) * (hd // 32) + i // 64 * 2 + i // 8 % 2
    v_at = base + 8 * hd + ((i // 32 * 16 + i % 16) * 4 + p // 16 % 2 * 2 + p // 4 % 2) * 4 + i // 16 % 2 * 2 + p // 32
    k_scale = base + 16 * hd + g * 64 + p
    return (k_at, shift(i % 8), k_scale), (v_at, shift(p // 8 % 2 * 4 + p % 4), k_scale + hd)


def _write_and_read(st):
    rows = st["pos"][:, None].long() + torch.arange(st["M"], device="cuda")
    q, k = rotate(st["q"], st["rope"], rows), rotate(st["k"], st["rope"], rows)
    words = st["cache"].view(-1).view(torch.int32)
    out = [q]
    places = _places(rows, st["hd"], st["Hkv"], st["cache"].shape[2])
    for x, (at, shift, scale_at) in zip((k, st["v"]), places):
        c, z, h = quantise(x)
        # a dword's eight codes change by what each differs by: whole numbers, so the order is free
        words.index_add_(0, at.flatten(), ((c - ((words[at] >> shift) & 15)) << shift).to(torch.int32).flatten())
        words[scale_at.expand_as(z)] = scale_bits(z, h)
    for at, shift, scale_at in places:
        scale, c = words[scale_at][..., None], (words[at] >> shift) & 15
        z, h = (scale & -65536).view(torch.float32), (scale << 16).view(torch.float32)
        out.append((z + h * (2 * c.unflatten(-1, (-1, 64)) - 15)).flatten(-2).transpose(1, 2).contiguous())
    return tuple(out)


def _attend(st):
    q, (K, V) = st["q"], unpack(st["cache"])
    B, M, heads, hd = q.shape
    n, G = st["Hkv"], heads // st["Hkv"]
    rows = q.view(B, M, n, G, hd).transpose(1, 2).reshape(B, n, M * G, hd)
    s = rows @ K.transpose(2, 3) / math.sqrt(hd)
    last = (st["pos"][:, None] + torch.arange(M, device="cuda")).repeat_interleave(G, 1)
    s = s.masked_fill(torch.arange(K.shape[2], device="cuda") > last[:, None, :, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = (e @ V) / e.sum(-1, keepdim=True)
    return o.view(B, n, M, G, hd).transpose(1, 2).reshape(B, M, heads, hd)


def run(st):
    if own:
        hip = _backend()
        if st["kind"] == "read":
            return hip.kv4_read(st["cache"], st["pos"], st["M"])
        if st["kind"] == "write":
            q = hip.kv4_append(st["q"], st["k"], st["v"], st["cache"], st["rope"], st["pos"])
            return (q, *hip.kv4_read(st["cache"], st["pos"], st["M"]))
        return hip.kv4_attention(st["q"], st["cache"], st["pos"])
    if st["kind"] == "read":
        return tuple(x[:, :, :st["M"]].contiguous() for x in unpack(st["cache"]))
    return _write_and_read(st) if st["kind"] == "write" else _attend(st)


def _backend():
    if "rotor-rag_amd" not in sys.path:
        sys.path.insert(0, "rotor-rag_amd")
    from rotor.gpu_layers import get_gpu, last_error

    hip = get_gpu()
    if hip is None:
        raise RuntimeError(last_error())
    return hip


# ---- the definition, in 64 bits ----------------------------------------------------------


def _held(x):
    """What the cache holds of one group after another: x float64 [N, 64] (fp32 numbers) -> float64."""
    lo, hi = x.min(1).values, x.max(1).values
    bf16 = lambda t: t.to(torch.float32).to(torch.bfloat16).to(torch.float64)[:, None]  # noqa: E731
    z, h = bf16(hi / 2 + lo / 2), bf16((hi / 2 - lo / 2) / 15)
    level = ((x - z) / torch.where(h > 0, h, torch.inf) + 15) / 2
    return z + h * (2 * level.round().clamp(0, 15) - 15)


def _cached(words, b, n, first, last, hd):
    """Positions [first, last) of head n of sequence b of the cache as dwords [B, Hkv, blocks, 18 hd]:
    K and V float64 [last - first, hd], element by element from the block's description."""
    p = torch.arange(first, last, device=words.device)[:, None]
    d = torch.arange(hd, device=words.device)[None]
    block = words[b, n].to(torch.int64)
    j, P = p // 64, p % 64
    kw = block[j, P * hd // 8 + (d % 64 // 16) * 2 * (hd // 64) + d // 64 * 2 + d % 16 // 8]
    vw = block[j, 8 * hd + (d // 32 * 16 + d % 16) * 16 + (P % 32 // 16 * 2 + P % 8 // 4) * 4 + d % 32 // 16 * 2 + P // 32]
    found = []
    for word, e, at in ((kw, d % 8, 16 * hd), (vw, P % 16 // 8 * 4 + P % 4, 17 * hd)):
        c = (word >> (e // 2 * 4 + e % 2 * 16)) & 15
        scale = block[j, at + d // 64 * 64 + P]
        z, h = (((scale >> s & 65535) << 16).to(torch.int32).view(torch.float32).double() for s in (16, 0))
        found.append(z + h * (2 * c - 15))
    return found


def exact(case, seed):
    st = prepare(case, seed)
    B, M, Hkv, hd = case["B"], case["M"], case["Hkv"], case["hd"]
    pos = _positions(case)
    if case["kind"] == "write":
        angle = torch.stack([st["rope"][p:p + M] for p in pos]).double()  # [B, M, hd / 2, 2]
        turn = torch.view_as_complex(angle)[:, :, None]
        turned = []
        for x in (st["q"], st["k"]):
            y = torch.complex(*x.double().chunk(2, -1)) * turn
            turned.append(torch.cat([y.real, y.imag], -1))
        k = turned[1].float().double()  # what is quantised is the key as an fp32 number
        back = lambda x: _held(x.reshape(-1, 64)).view(x.shape).transpose(1, 2).contiguous()  # noqa: E731
        return (turned[0], back(k), back(st["v"].double()))
    words = st["cache"].view(torch.int32)
    if case["kind"] == "read":
        K, V = (torch.empty((B, Hkv, M, hd), dtype=torch.float64, device="cuda") for _ in range(2))
        for b in range(B):
            for n in range(Hkv):
                K[b, n], V[b, n] = _cached(words, b, n, 0, M, hd)
        return K, V
    G = case["H"] // Hkv
    o = torch.empty((B, M, Hkv, G, hd), dtype=torch.float64, device="cuda")
    q = st["q"].double().view(B, M, Hkv, G, hd)
    for b in range(B):
        seen = torch.arange(pos[b] + M, device="cuda")[None] <= pos[b] + torch.arange(M, device="cuda")[:, None]
        for n in range(Hkv):
            K, V = _cached(words, b, n, 0, pos[b] + M, hd)
            for g in range(G):
                s = torch.where(seen, q[b, :, n, g] @ K.T.contiguous() / hd ** 0.5, -torch.inf)
                o[b, :, n, g] = torch.softmax(s, -1) @ V
    return o.view(B, M, Hkv * G, hd)
