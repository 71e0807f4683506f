"""The paged KV cache without a GPU: sizes, every refusal of the C ABI and of the Python entry points (all decided before the
device is touched), and the angles scaled for long contexts."""
import ctypes
import math

import numpy as np
import pytest

from oracle import paged_oracle as PO

RT_EINVAL = -1


@pytest.fixture(scope="module")
def lib():
    from rotor import _hip

    return _hip.load()


def test_structures_match_the_header(tmp_path):
    """The packed forms have the size and the offsets of the header's structures."""
    import subprocess
    from pathlib import Path

    from rotor import _hip

    fields = ["cache", "kv_stride", "page_stride", "table", "lens", "type", "pages", "Hkv", "page", "hd", "B", "P"]
    new = ["q", "k", "v", "rope", "pos", "counts", "rope_rows", "rotary", "interleaved", "M", "H"]
    header = Path(__file__).resolve().parents[1] / "include" / "rotor_hip.h"
    code = f'#include "{header}"\n#include <stdio.h>\nint main(void) {{ printf("%zu %zu", sizeof(rt_pages), sizeof(rt_paged_new));\n'
    code += "".join(f'printf(" %zu", offsetof({s}, {f}));\n' for s, fs in (("rt_pages", fields), ("rt_paged_new", new)) for f in fs)
    (tmp_path / "a.c").write_text(code + "return 0; }\n")
    subprocess.run(["gcc", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    assert got[:2] == [_hip.PAGES.size, _hip.PAGED_NEW.size]
    a = _hip.PAGES.unpack(bytes(i % 251 for i in range(got[0])))
    for at, value, size in zip(got[2:], a, [8] * 5 + [4] * 7):
        assert value == int.from_bytes(bytes(i % 251 for i in range(at, at + size)), "little", signed=False)
    b = _hip.PAGED_NEW.unpack(bytes(i % 251 for i in range(got[1])))
    for at, value, size in zip(got[2 + len(a):], b, [8] * 6 + [4] * 5):
        assert value == int.from_bytes(bytes(i % 251 for i in range(at, at + size)), "little", signed=False)


# A refused call returns before it looks into the context or at the device, so any non-NULL pointers do.
_CTX = ctypes.create_string_buffer(4096)
PTR = ctypes.addressof(_CTX) + 15 & ~15
ODD = PTR + 4
ROWS = 5 * 64 * 128
CACHE = dict(cache=PTR, kv_stride=100 * ROWS, page_stride=ROWS, table=PTR, lens=PTR, type=1, pages=100, Hkv=5, page=64, hd=128, B=3, P=40)
NEW = dict(q=PTR, k=PTR, v=PTR, rope=PTR, pos=PTR, counts=0, rope_rows=640, rotary=128, interleaved=0, M=1, H=20)
CALLS = ["append", "attention", "step", "evict"]


def call(lib, name, cache=CACHE, new=NEW, ctx=PTR, **kw):
    from rotor import _hip

    c = _hip.PAGES.pack(*cache.values()) if cache is not None else None
    n = _hip.PAGED_NEW.pack(*new.values()) if new is not None else None
    a = dict(out=PTR, weights=PTR, slots=64 * 40, ws=PTR, bytes=1 << 40, q=PTR, H=20, keep=100, recent=10, table=PTR + 64, P=10, kept=PTR,
             lens=PTR + 128, left=PTR + 256)
    assert set(kw) <= set(a)
    a.update(kw)
    if name == "append":
        return lib.rt_paged_append(ctx, c, n, a["out"])
    if name == "attention":
        return lib.rt_paged_attention(ctx, c, a["q"], a["H"], a["weights"], a["slots"], a["out"], a["ws"], a["bytes"])
    if name == "step":
        return lib.rt_paged_step(ctx, c, n, a["weights"], a["slots"], a["out"], a["ws"], a["bytes"])
    return lib.rt_paged_evict(ctx, c, a["weights"], a["slots"], a["keep"], a["recent"], a["table"], a["P"], a["kept"], a["lens"], a["left"],
                              a["ws"], a["bytes"])


def refused(lib, name, match, **kw):
    assert call(lib, name, **kw) == RT_EINVAL, kw
    text = lib.rt_last_error().decode()
    assert text.startswith("rt_paged_" + name) and match in text, text


@pytest.mark.parametrize("name", CALLS)
def test_refused_caches(lib, name):
    refused(lib, name, "NULL", ctx=None)
    refused(lib, name, "NULL", cache=None)
    for field in ("cache", "table", "lens"):
        refused(lib, name, "NULL", cache=dict(CACHE, **{field: 0}))
    refused(lib, name, "aligned", cache=dict(CACHE, cache=ODD))
    for bad in [dict(type=3), dict(type=-1), dict(hd=32), dict(hd=256), dict(hd=0), dict(page=8), dict(page=512), dict(page=48),
                dict(page=0), dict(page=-16), dict(pages=0), dict(pages=-1), dict(Hkv=0), dict(Hkv=-5), dict(B=0), dict(B=-1), dict(B=1 << 23),
                dict(P=0), dict(P=-1), dict(P=16385), dict(P=2 ** 31 - 1)]:
        refused(lib, name, "layout", cache=dict(CACHE, **bad))
    for bad in [dict(page_stride=ROWS - 8), dict(page_stride=0), dict(page_stride=-ROWS), dict(kv_stride=0), dict(kv_stride=-ROWS),
                dict(kv_stride=ROWS - 8), dict(page_stride=2 ** 62), dict(kv_stride=2 ** 62)]:
        refused(lib, name, "stride", cache=dict(CACHE, **bad))
    for bad in [dict(kv_stride=50 * ROWS), dict(kv_stride=100 * ROWS - 8), dict(kv_stride=ROWS), dict(kv_stride=ROWS, page_stride=2 * ROWS - 8)]:
        refused(lib, name, "overlap", cache=dict(CACHE, **bad))
    refused(lib, name, "aligned", cache=dict(CACHE, page_stride=ROWS + 4, kv_stride=200 * ROWS))
    refused(lib, name, "aligned", cache=dict(CACHE, kv_stride=100 * ROWS + 4))


@pytest.mark.parametrize("name", ["append", "step"])
def test_refused_tokens(lib, name):
    refused(lib, name, "NULL", new=None)
    refused(lib, name, "NULL", out=None)
    for field in ("q", "k", "v", "rope", "pos"):
        refused(lib, name, "NULL", new=dict(NEW, **{field: 0}))
        if field != "pos":
            refused(lib, name, "aligned", new=dict(NEW, **{field: ODD}))
    refused(lib, name, "aligned", out=ODD)
    for bad in [dict(M=0), dict(M=-1), dict(M=(1 << 20) + 1)]:
        refused(lib, name, "M", new=dict(NEW, **bad))
    for bad in [dict(rotary=0), dict(rotary=4), dict(rotary=132), dict(rotary=136), dict(rotary=-8), dict(rope_rows=0), dict(rope_rows=-1)]:
        refused(lib, name, "rotary", new=dict(NEW, **bad))
    for bad in [0, 21, -20, 5 * 1025, 5 << 18]:
        refused(lib, name, "layout", new=dict(NEW, H=bad))
    wide = dict(CACHE, Hkv=2048, page=16, hd=64, page_stride=1 << 30, kv_stride=1 << 38)
    refused(lib, name, "layout", cache=wide, new=dict(NEW, H=2048 * 513, rotary=64))
    if name == "step":
        refused(lib, name, "one token", new=dict(NEW, M=2))
        refused(lib, name, "one token", new=dict(NEW, counts=PTR))


@pytest.mark.parametrize("name", ["attention", "step"])
def test_refused_attention(lib, name):
    from rotor import _hip

    refused(lib, name, "NULL", out=None)
    refused(lib, name, "aligned", out=ODD)
    refused(lib, name, "slots", slots=64 * 40 - 1)
    refused(lib, name, "slots", slots=0)
    c = _hip.PAGES.pack(*CACHE.values())
    for weights in (0, 1):
        need = lib.rt_paged_attention_workspace(c, 20, weights)
        assert need > 0
        kw = dict(weights=PTR if weights else None)
        for bad in (dict(bytes=need - 1), dict(ws=None), dict(ws=ODD)):
            refused(lib, name, "workspace", **kw, **bad)
    if name == "attention":
        refused(lib, name, "NULL", q=None)
        refused(lib, name, "aligned", q=ODD)
        for bad in (0, 21, -20, 5 * 1025):
            refused(lib, name, "layout", H=bad)


def test_refused_evictions(lib):
    for field in ("weights", "table", "kept", "lens", "left"):
        refused(lib, "evict", "NULL", **{field: None})
    for bad in [dict(keep=0), dict(keep=-1), dict(recent=-1), dict(recent=101), dict(keep=641), dict(P=0), dict(P=-1), dict(P=16385)]:
        refused(lib, "evict", "keep", **bad)
    refused(lib, "evict", "slots", slots=64 * 40 - 1)
    for bad in [dict(left=PTR), dict(table=PTR), dict(lens=PTR)]:
        refused(lib, "evict", "other memory", **bad)


def test_refused_eviction_workspaces(lib):
    from rotor import _hip

    small, large = dict(CACHE, P=512), dict(CACHE, P=513)  # 32768 slots, and a page more
    assert lib.rt_paged_evict_workspace(_hip.PAGES.pack(*small.values())) == 0
    need = lib.rt_paged_evict_workspace(_hip.PAGES.pack(*large.values()))
    assert need > 0 and lib.rt_paged_evict_workspace(_hip.PAGES.pack(*dict(large, hd=32).values())) == 0
    for bad in (dict(bytes=need - 1), dict(ws=None), dict(ws=ODD)):
        refused(lib, "evict", "workspace", cache=large, slots=1 << 20, **bad)


def test_workspace_sizes(lib):
    from rotor import _hip

    def size(H=20, weights=0, **kw):
        return lib.rt_paged_attention_workspace(_hip.PAGES.pack(*dict(CACHE, **kw).values()), H, weights)

    assert size(B=1, P=1) == 0                          # one split, and nothing to keep
    assert size(B=1, P=1, weights=1) >= 4 * 20 * 64     # the scores
    assert size(B=1, P=2048) > 0
    assert size(B=5000, P=2048) == 0                    # more heads than any launch has places for: a piece each
    assert size(B=256, P=16384, weights=1) >= 4 * 256 * 20 * (1 << 20)  # 64-bit
    for bad in [dict(H=21), dict(hd=32), dict(P=0), dict(pages=0)]:
        assert size(**bad) == 0


@pytest.fixture()
def ops(lib):
    """The Python entry points on CPU tensors: every refusal comes before the library is called."""
    torch = pytest.importorskip("torch")
    from rotor.gpu_ternary import HIPTernaryOps

    o = HIPTernaryOps.__new__(HIPTernaryOps)
    o.lib, o.device, o.device_index, o.ctx = lib, torch.device("cpu"), -1, None
    return o


def test_python_cache(ops):
    import torch

    c = ops.paged_cache(5, 128, 7)
    assert tuple(c.shape) == (2, 7, 5, 64, 128) and c.dtype == torch.bfloat16 and c.isnan().all()
    assert ops.paged_cache(1, 64, 1, page=16, dtype=torch.float32).isnan().all()
    for bad in [dict(head_dim=96), dict(page=8), dict(page=48), dict(page=512), dict(dtype=torch.float64), dict(dtype=torch.int8),
                dict(n_pages=0), dict(n_kv_heads=0)]:
        with pytest.raises(ValueError, match="paged_cache"):
            ops.paged_cache(**{**dict(n_kv_heads=2, head_dim=64, n_pages=3, page=32), **bad})


@pytest.fixture()
def given(ops):
    import torch

    f = lambda *s: torch.zeros(s)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(cache=ops.paged_cache(2, 64, 9, 16), table=i(3, 4), lens=i(3), q=f(3, 1, 6, 64), k=f(3, 1, 2, 64), v=f(3, 1, 2, 64),
                rope=f(100, 32, 2), pos=i(3), weights=f(3, 2, 64), keep=20, recent=4, new_table=i(3, 2))


def python_call(ops, name, a, **kw):
    a = {**a, **kw}
    tokens = [a[x] for x in ("q", "k", "v", "cache", "table", "lens", "rope", "pos")]
    if name == "append":
        return ops.paged_append(*tokens, counts=a.get("counts"), q_out=a.get("out"))
    if name == "attention":
        return ops.paged_attention(a["q"], a["cache"], a["table"], a["lens"], weights=a["weights"], out=a.get("out"))
    if name == "step":
        return ops.paged_step(*tokens, weights=a["weights"], out=a.get("out"))
    return ops.paged_evict(a["cache"], a["table"], a["lens"], a["weights"], a["keep"], a["recent"], a["new_table"])


@pytest.mark.parametrize("name", CALLS)
def test_python_refusals(ops, given, name):
    import torch

    f = lambda *s: torch.zeros(s)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    c = given["cache"]
    bad = [dict(cache=x) for x in (c.double(), c.to(torch.int16), c[0], c[:1], c[..., :32], c.transpose(2, 3), c[:, :, :, ::2],
                                   c.transpose(3, 4).contiguous().transpose(3, 4))]
    bad += [dict(table=x) for x in (i(3, 4).long(), i(2, 4), i(12), i(3, 8)[:, ::2], i(4, 3).T)]
    bad += [dict(lens=x) for x in (i(3).long(), i(2), i(6)[::2], i(3, 1))]
    if name in ("append", "step"):
        bad += [dict(q=x) for x in (f(2, 1, 6, 64), f(3, 1, 5, 64), f(3, 1, 6, 128), f(3, 6, 64), f(3, 0, 6, 64))]
        bad += [{n: x} for n in "kv" for x in (f(3, 1, 1, 64), f(3, 2, 2, 64), f(3, 2, 64))]
        bad += [dict(rope=x) for x in (f(100, 32), f(100, 30, 2), f(100, 36, 2), f(100, 32, 3), f(0, 32, 2), f(100, 0, 2))]
        bad += [dict(pos=x) for x in (i(3).long(), i(2), i(6)[::2])]
    if name == "append":
        bad += [dict(counts=x) for x in (i(3).long(), i(2), i(6)[::2])]
    if name == "attention":
        bad += [dict(q=x) for x in (f(2, 1, 6, 64), f(3, 1, 5, 64), f(3, 2, 6, 64), f(3, 6, 64))]
    if name != "append":
        bad += [dict(weights=x) for x in (f(3, 2, 63), f(2, 2, 64), f(3, 1, 64), f(3, 2, 64).double(), f(3, 2, 128)[..., ::2], f(6, 64))]
    if name == "evict":
        bad += [dict(new_table=x) for x in (i(3, 2).long(), i(2, 2), i(3), i(3, 4)[:, ::2], i(3, 1), given["table"], given["table"][:, :])]
        bad += [dict(keep=0), dict(keep=-1), dict(keep=33), dict(recent=-1), dict(recent=21)]
    else:
        q = given["q"]
        bad += [dict(out=x) for x in (f(3, 1, 6, 32), q.double(), f(3, 1, 12, 64)[:, :, ::2])]
    for kw in bad:
        with pytest.raises(ValueError, match="paged_" + name):
            python_call(ops, name, given, **kw)
    if name == "step":
        with pytest.raises(ValueError, match="one token"):
            python_call(ops, name, given, q=f(3, 2, 6, 64), k=f(3, 2, 2, 64), v=f(3, 2, 2, 64))
    if name == "evict":
        with pytest.raises(TypeError):
            python_call(ops, name, given, keep=2.5)


def test_python_outputs_apart(ops, given):
    """Outputs in the memory of what a call reads (q itself may be the output)."""
    import torch

    big = torch.zeros(4, 1, 6, 64)
    flat = big.view(-1)
    n = given["q"].numel()
    for name in ("append", "step"):
        for kw in (dict(q=big[1:], out=big[:3]), dict(k=flat[:384].view(3, 1, 2, 64), out=big[:3]), dict(rope=flat[:64].view(1, 32, 2), out=big[:3]),
                   dict(pos=flat.view(torch.int32)[4:7], out=big[:3]), dict(lens=flat.view(torch.int32)[4:7], out=big[:3]),
                   dict(table=flat.view(torch.int32)[4:16].view(3, 4), out=big[:3]),
                   dict(out=given["cache"].view(-1)[:2 * n].view(torch.float32).view(3, 1, 6, 64))):
            with pytest.raises(ValueError, match="share memory"):
                python_call(ops, name, given, **kw)
    for name in ("attention", "step"):
        for kw in (dict(q=big[1:], out=big[:3], weights=None), dict(out=big[:3], weights=flat[:384].view(3, 2, 64)), dict(q=big[:3], weights=flat[:384].view(3, 2, 64)),
                   dict(weights=given["cache"].view(-1)[:768].view(torch.float32).view(3, 2, 64))):
            with pytest.raises(ValueError, match="share memory"):
                python_call(ops, name, given, **kw)


# ---- angles ------------------------------------------------------------------------------


def test_rope_scaling():
    from rotor.bitnet_model import config_from_hf, rope_table

    plain = rope_table(500, 64, 10000.0)
    assert np.array_equal(rope_table(500, 64, 10000.0, {"rope_type": "default"}), plain)
    linear = rope_table(500, 64, 10000.0, {"type": "linear", "factor": 4.0})
    assert np.array_equal(linear[::4], plain[:125])
    ntk = rope_table(500, 64, 10000.0, {"rope_type": "ntk", "factor": 4.0})
    assert np.array_equal(ntk[:, 0], plain[:, 0])                        # the fastest pair as it is
    assert np.allclose(ntk[:, -1], linear[:, -1], atol=1e-6)             # the slowest like linear
    yarn = rope_table(3000, 64, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048})
    grow = 0.1 * math.log(4.0) + 1
    assert np.allclose(np.hypot(yarn[..., 0], yarn[..., 1]), grow, atol=1e-6)
    turns = 2048 * 10000.0 ** (-np.arange(32) / 32) / (2 * math.pi)
    fast, slow = turns > 34, turns < 0.9
    assert fast.any() and slow.any()
    a = np.arctan2(yarn[1, :, 1], yarn[1, :, 0])
    b = np.arctan2(plain[1, :, 1], plain[1, :, 0])
    assert np.allclose(a[fast], b[fast], rtol=1e-6) and np.allclose(a[slow], b[slow] / 4, rtol=1e-5)
    between = ~fast & ~slow
    assert ((a[between] <= b[between] * (1 + 1e-6)) & (a[between] >= b[between] / 4 * (1 - 1e-6))).all()
    one = rope_table(10, 64, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048, "attention_factor": 1.0})
    assert np.allclose(np.hypot(one[..., 0], one[..., 1]), 1.0, atol=1e-6)
    for bad in ({"rope_type": "other", "factor": 2.0}, {"rope_type": "linear", "factor": 0.0}, {"rope_type": "yarn", "factor": 2.0}, {"factor": 2.0},
                {"rope_type": "ntk", "factor": float("nan")}):
        with pytest.raises(ValueError, match="rope_scaling"):
            rope_table(10, 64, 10000.0, bad)
    cfg = dict(vocab_size=64, hidden_size=256, num_hidden_layers=1, num_attention_heads=2, intermediate_size=256)
    assert "rope_scaling" not in config_from_hf(dict(cfg, rope_scaling=None))
    assert config_from_hf(dict(cfg, rope_scaling={"rope_type": "linear", "factor": 2.0}))["rope_scaling"]["factor"] == 2.0


# ---- the oracle's own properties -----------------------------------------------------------


def test_oracle():
    import torch

    cache = torch.randn(2, 5, 2, 16, 64)
    table = torch.tensor([[3, 1], [0, 4]], dtype=torch.int32)
    lens = torch.tensor([20, 0], dtype=torch.int32)
    o, w, _, _ = PO.attend(torch.randn(2, 1, 4, 64), cache, table, lens)
    assert torch.allclose(w.sum(-1), torch.tensor([[2.0, 2.0], [0.0, 0.0]], dtype=torch.float64)) and (o[1] == 0).all()
    kept = PO.evict(cache, table, lens, torch.ones(2, 2, 32), 7, 3)
    assert kept == [[[0, 1, 2, 3, 17, 18, 19]] * 2, [[], []]]
    x = torch.randn(3, 64, dtype=torch.float64)
    angles = torch.tensor([[0.0, 1.0]] * 4)
    y = PO.rotate(x, angles, True)
    assert torch.equal(y[:, 0], -x[:, 1]) and torch.equal(y[:, 1], x[:, 0]) and torch.equal(y[:, 8:], x[:, 8:])
    y = PO.rotate(x, angles, False)
    assert torch.equal(y[:, 0], -x[:, 4]) and torch.equal(y[:, 4], x[:, 0])
