"""The 4-bit KV cache without a GPU: the definition's own properties, the sizes, and every
refusal of the C ABI and of the Python entry points (all decided before the device is touched)."""
import ctypes

import numpy as np
import pytest

from oracle import kv4_oracle as K4

RT_EINVAL = -1


@pytest.fixture(scope="module")
def lib():
    from rotor import _hip

    return _hip.load()


@pytest.mark.parametrize("scale,shift", [(1.0, 0.0), (1e-20, 0.0), (1e20, 0.0), (0.01, 3.0), (5.0, -40.0), (1e-44, 0.0)])
def test_definition_error_bound(scale, shift):
    """|x - value| <= h + 15 h 2^-8 + |z| 2^-8: half a step (h) inside the levels' range; the range itself
    may end early by the roundings of h and z (2^-9 relative each in the normal range, doubled for the
    two rounding steps), and by a bf16 subnormal's half step (2^-134) times 16 below it."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((40, 128)) * scale + shift).astype(np.float32)
    c, z, h = K4.quantise(x)
    assert c.min() >= 0 and c.max() <= 15
    rep = lambda a: np.repeat(a, 64, -1)  # noqa: E731
    bound = rep(h) * (1 + 15 * 2.0 ** -8) + np.abs(rep(z)) * 2.0 ** -8 + 16 * 2.0 ** -134
    v = rep(z) + rep(h) * (2 * c - 15)
    assert (np.abs(x.astype(np.float64) - v) <= bound).all()


def test_definition_special_groups():
    x = np.zeros((6, 64), np.float32)
    x[1] = 2.5                      # constant: exact where bf16 holds it
    x[2, 7] = np.nan
    x[3, 0] = -np.inf
    x[4] = np.float32(3.4e38)       # rounds past bf16's largest
    x[5, ::2], x[5, 1::2] = 3e38, -3e38  # the extremes' difference passes fp32
    v = K4.held(x)
    assert (v[0] == 0).all() and (v[1] == 2.5).all()
    assert np.isnan(v[2:5]).all()
    assert np.isfinite(v[5]).all() and np.allclose(v[5], x[5], rtol=2 ** -7)


def test_codes_ties_to_even():
    # z = 0, h = 1: x = 2 c - 15 + 1 lies half way between levels c and c + 1
    x = np.zeros((1, 64), np.float32)
    x[0, 0], x[0, 1] = -15, 15
    x[0, 2:16] = np.arange(-14, 14, 2)
    c, z, h = K4.quantise(x)
    assert z[0, 0] == 0 and h[0, 0] == 1
    assert list(c[0, 2:16]) == [2 * ((i + 1) // 2) for i in range(14)]


def test_bytes(lib):
    assert lib.rt_kv4_bytes(1, 5, 128, 2048) == 5 * 32 * 9216
    assert lib.rt_kv4_bytes(3, 2, 64, 65) == 3 * 2 * 2 * 4608
    assert lib.rt_kv4_bytes(64, 8, 128, 1 << 20) == 64 * 8 * 16384 * 9216  # 77 GB: 64-bit
    for bad in [(0, 5, 128, 64), (1, 0, 128, 64), (1, 5, 96, 64), (1, 5, 128, 0), (1, 5, 128, (1 << 20) + 1),
                (1 << 20, 32, 64, 64), (-1, 5, 128, 64)]:
        assert lib.rt_kv4_bytes(*bad) == 0


def test_workspace_sizes(lib):
    """Nothing for calls that fill the GPU by themselves, something for one token, 0 for refused sizes."""
    assert lib.rt_kv4_attention_workspace(1, 1, 20, 5, 128, 131072) > 0
    assert lib.rt_kv4_attention_workspace(1, 1, 20, 5, 128, 64) == 0
    assert lib.rt_kv4_attention_workspace(1, 1, 20, 5, 128, 640) == 0  # few keys a wave as it is
    assert lib.rt_kv4_attention_workspace(64, 512, 20, 5, 128, 4096) == 0
    for bad in [(1, 1, 21, 5, 128, 64), (1, 65, 20, 5, 128, 64), (1, 0, 20, 5, 128, 64), (1, 1, 20, 5, 32, 64),
                (1, 1, 0, 5, 128, 64), (1, 1, 1025, 1, 64, 64)]:
        assert lib.rt_kv4_attention_workspace(*bad) == 0


# A refused call returns before it looks into the context or at the device, so any non-NULL pointers do.
_CTX = ctypes.create_string_buffer(4096)
P = ctypes.addressof(_CTX) + 15 & ~15
ODD = P + 4
GOOD = dict(B=1, M=1, H=20, Hkv=5, hd=128, Lmax=640)


def _append(lib, ctx=P, q=P, k=P, v=P, rope=P, cache=P, q_out=P, pos=P, **kw):
    a = {**GOOD, **kw}
    return lib.rt_kv4_append(ctx, q, k, v, rope, cache, q_out, a["B"], a["M"], a["H"], a["Hkv"], a["hd"], a["Lmax"], pos)


def _read(lib, ctx=P, cache=P, k=P, v=P, pos=P, **kw):
    a = {**GOOD, **kw}
    return lib.rt_kv4_read(ctx, cache, k, v, a["B"], a["M"], a["Hkv"], a["hd"], a["Lmax"], pos)


def _attend(lib, ctx=P, q=P, cache=P, out=P, pos=P, ws=P, ws_bytes=1 << 30, **kw):
    a = {**GOOD, **kw}
    return lib.rt_kv4_attention(ctx, q, cache, out, a["B"], a["M"], a["H"], a["Hkv"], a["hd"], a["Lmax"], pos, ws,
                                ws_bytes)


def _step(lib, ctx=P, q=P, k=P, v=P, rope=P, cache=P, out=P, pos=P, ws=P, ws_bytes=1 << 30, **kw):
    a = {**GOOD, **kw}
    return lib.rt_kv4_step(ctx, q, k, v, rope, cache, out, a["B"], a["H"], a["Hkv"], a["hd"], a["Lmax"], pos, ws, ws_bytes)


BAD_SIZES = [dict(B=0), dict(B=-1), dict(M=0), dict(M=641), dict(Hkv=0), dict(Hkv=-5), dict(hd=32), dict(hd=256),
             dict(hd=0), dict(Lmax=0), dict(Lmax=(1 << 20) + 1), dict(B=1 << 22), dict(B=1 << 30, Hkv=4)]


@pytest.mark.parametrize("call,bufs", [(_append, ["ctx", "q", "k", "v", "rope", "cache", "q_out", "pos"]),
                                       (_read, ["ctx", "cache", "k", "v", "pos"]),
                                       (_attend, ["ctx", "q", "cache", "out", "pos"]),
                                       (_step, ["ctx", "q", "k", "v", "rope", "cache", "out", "pos"])])
def test_refusals(lib, call, bufs):
    who = {"_append": "rt_kv4_append", "_read": "rt_kv4_read", "_attend": "rt_kv4_attention",
           "_step": "rt_kv4_step"}[call.__name__]
    for name in bufs:
        assert call(lib, **{name: None}) == RT_EINVAL
        assert who in lib.rt_last_error().decode() and "NULL" in lib.rt_last_error().decode()
        if name not in ("ctx", "pos"):
            assert call(lib, **{name: ODD}) == RT_EINVAL
            assert who in lib.rt_last_error().decode() and "aligned" in lib.rt_last_error().decode()
    for bad in BAD_SIZES:
        if call is _step and "M" in bad:
            continue
        assert call(lib, **bad) == RT_EINVAL, bad
        assert who in lib.rt_last_error().decode()
    if call is not _read:
        for bad in [dict(H=0), dict(H=21), dict(H=-20), dict(H=1025, Hkv=1)]:
            assert call(lib, **bad) == RT_EINVAL, bad
    if call is _step:
        assert call(lib, H=17, Hkv=1) == RT_EINVAL and "H / Hkv" in lib.rt_last_error().decode()


def test_attention_refuses_small_workspaces(lib):
    need = lib.rt_kv4_attention_workspace(1, 1, 20, 5, 128, 4096)
    assert need > 0
    for bad in [dict(ws=None, ws_bytes=0), dict(ws_bytes=need - 1), dict(ws=ODD, ws_bytes=need)]:
        for call in (_attend, _step):
            assert call(lib, Lmax=4096, **bad) == RT_EINVAL
            assert "workspace" in lib.rt_last_error().decode()


@pytest.fixture()
def ops(lib):
    """The Python entry points on CPU tensors: every refusal comes before the library is called."""
    torch = pytest.importorskip("torch")
    from rotor.gpu_ternary import HIPTernaryOps

    o = HIPTernaryOps.__new__(HIPTernaryOps)
    o.lib, o.device, o.device_index, o.ctx = lib, torch.device("cpu"), -1, None
    return o


def test_python_cache_shapes(ops):
    c = ops.kv4_cache(5, 128, 130, batch=3)
    assert tuple(c.shape) == (3, 5, 3, 9216)
    assert c.numel() == ops.lib.rt_kv4_bytes(3, 5, 128, 130)
    for bad in [(5, 96, 64), (0, 128, 64), (5, 128, 0), (5, 128, (1 << 20) + 1)]:
        with pytest.raises(ValueError, match="kv4_cache"):
            ops.kv4_cache(*bad)


def test_python_refusals(ops):
    import torch

    f = lambda *s: torch.zeros(s)  # noqa: E731
    cache, pos, rope = ops.kv4_cache(2, 64, 100, batch=3), torch.zeros(3, dtype=torch.int32), f(100, 32, 2)
    q, kv = f(3, 4, 6, 64), f(3, 4, 2, 64)
    bad_caches = [cache[:, :, :, :100], cache.float(), cache[0], cache.transpose(0, 1)]
    bad_pos = [pos.long(), pos[:2], torch.zeros(6, dtype=torch.int32)[::2], pos[None]]
    for c, p in [(c, pos) for c in bad_caches] + [(cache, p) for p in bad_pos]:
        for call in (lambda: ops.kv4_append(q, kv, kv, c, rope, p), lambda: ops.kv4_read(c, p, 5),
                     lambda: ops.kv4_attention(q, c, p)):
            with pytest.raises(ValueError):
                call()
    for n in (0, 64, 129, -1):  # positions that are not those of two blocks
        with pytest.raises(ValueError, match="max_len"):
            ops.kv4_attention(q, cache, pos, max_len=n)
    for args in [(q[..., :32], kv, kv, rope), (q[:2], kv, kv, rope), (q[0], kv, kv, rope), (f(3, 4, 5, 64), kv, kv, rope),
                 (q, kv[:, :3], kv, rope), (q, kv, f(3, 4, 1, 64), rope), (q, kv, kv, rope[:64]), (q, kv, kv, rope[..., 0]),
                 (f(3, 0, 6, 64), f(3, 0, 2, 64), f(3, 0, 2, 64), rope)]:
        with pytest.raises(ValueError, match="kv4_append"):
            ops.kv4_append(*args[:3], cache, args[3], pos)
    one, kv1 = q[:, :1].contiguous(), kv[:, :1].contiguous()
    for args in [(q, kv, kv, rope), (one[..., :32], kv1, kv1, rope), (one, kv, kv1, rope), (one, kv1, kv1, rope[:64]),
                 (f(3, 1, 34, 64), kv1, kv1, rope)]:
        with pytest.raises(ValueError, match="kv4_step"):
            ops.kv4_step(*args[:3], cache, args[3], pos)
    for n in (0, -1, 129):
        with pytest.raises(ValueError, match="length"):
            ops.kv4_read(cache, pos, n)
    with pytest.raises(ValueError, match="rope"):
        ops.kv4_append(q, kv, kv, cache, rope[:99], pos, max_len=100)
    with pytest.raises(ValueError, match="output"):
        ops.kv4_append(q, kv, kv, cache, rope, pos, q_out=f(3, 4, 6, 32))
    for bad in (q[:2], q[0], f(3, 4, 5, 64), f(3, 4, 6, 128), f(3, 0, 6, 64)):
        with pytest.raises(ValueError, match="kv4_attention"):
            ops.kv4_attention(bad, cache, pos)
    for out in (f(3, 4, 6, 32), q.double(), q.transpose(1, 2)):
        with pytest.raises(ValueError, match="output"):
            ops.kv4_attention(q, cache, pos, out=out)
    # outputs in another argument's memory (q itself may be one)
    both = f(4, 4, 6, 64)
    for call in (lambda: ops.kv4_append(both[1:], kv, kv, cache, rope, pos, q_out=both[:3]),
                 lambda: ops.kv4_append(q, both.view(-1)[:kv.numel()].view(kv.shape), kv, cache, rope, pos, q_out=both[:3]),
                 lambda: ops.kv4_append(q, kv, both.view(-1)[-kv.numel():].view(kv.shape), cache, rope, pos, q_out=both[1:]),
                 lambda: ops.kv4_step(one, kv1, kv1, cache, rope, pos, out=rope.view(-1)[:one.numel()].view(one.shape)),
                 lambda: ops.kv4_attention(both[:3], cache, pos, out=both[1:]),
                 lambda: ops.kv4_attention(q, cache, pos, out=cache.view(-1)[:4 * q.numel()].view(torch.float32).view(q.shape))):
        with pytest.raises(ValueError, match="share memory"):
            call()
    with pytest.raises(TypeError):
        ops.kv4_read(cache, pos, 2.5)


def test_python_cache_is_nan_until_written(ops):
    """Every group of a new cache reads as NaN by the definition: z NaN, h 0."""
    for hd in (64, 128):
        words = ops.kv4_cache(3, hd, 130, batch=2).numpy().view(np.uint32)
        scales = words[..., 16 * hd:]
        z, h = ((x << np.uint32(16)).view(np.float32) for x in (scales >> np.uint32(16), scales & np.uint32(0xFFFF)))
        assert scales.size == 2 * 3 * 3 * 2 * hd and np.isnan(z).all() and (h == 0).all()


def test_config_file_keeps_the_cache_bits():
    from rotor.bitnet_model import config_from_hf

    cfg = dict(vocab_size=64, hidden_size=256, num_hidden_layers=1, num_attention_heads=2, intermediate_size=256)
    assert "kv_cache_bits" not in config_from_hf(cfg)
    assert config_from_hf(dict(cfg, kv_cache_bits=4))["kv_cache_bits"] == 4


def test_python_outputs_in_the_positions_memory(ops):
    """An output over pos would move the rows of the workgroups that come later."""
    import torch

    out = torch.zeros(2, 1, 2, 64)
    pos = out.view(torch.int32).view(-1)[64:66]
    cache, rope, kv = ops.kv4_cache(2, 64, 64, batch=2), torch.zeros(64, 32, 2), torch.zeros(2, 1, 2, 64)
    for call in (lambda: ops.kv4_append(kv, kv, kv, cache, rope, pos, q_out=out), lambda: ops.kv4_attention(kv, cache, pos, out=out),
                 lambda: ops.kv4_step(kv, kv, kv, cache, rope, pos, out=out), lambda: ops.kv4_attention(out, cache, pos, out=out)):
        with pytest.raises(ValueError, match="share memory"):
            call()
