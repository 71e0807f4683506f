"""Calls of the 4-bit KV cache that its documentation allows and that once went wrong."""
import numpy as np
import pytest

import test_gpu_kv4 as G
from oracle import kv4_oracle as K4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 4, 70])
def test_rows_past_the_angles(hip, M):
    """A cache of 100 positions (blocks for 128), angles for 100, and no max_len: rows from 100 on are not appended,
    and attention, which does not see the angles, gives NaN for them; the rows before are as with max_len."""
    import torch

    B, H, Hkv, hd, Lmax = 2, 4, 2, 128, 100
    q, k, v = G._inputs(M, B, Lmax, H, Hkv, hd)
    table = G._rope(Lmax, hd)
    old = torch.full((B, Hkv, 2, 72 * hd), 0x3C, dtype=torch.uint8, device="cuda")  # memory that was used before
    del old
    cache = hip.kv4_cache(Hkv, hd, Lmax, batch=B)
    (rope,) = G._cuda(table)
    hip.kv4_append(*G._cuda(q, k, v), cache, rope, G._pos([0, 0]))
    pos = G._pos([Lmax - (M + 1) // 2, Lmax])
    new = [x[:, :M] for x in G._inputs(M + 1, B, M, H, Hkv, hd)]
    rows = hip.kv4_append(*G._cuda(*new), cache, rope, pos)
    y = hip.kv4_attention(rows, cache, pos)
    n = (M + 1) // 2
    for b, first in enumerate((Lmax - n, Lmax)):  # positions 100..127 are in the blocks, those behind in no cache
        at = first + torch.arange(M)
        assert torch.isnan(y[b, (at >= Lmax) & (at < 128)]).all() and (y[b, at >= 128] == 0).all()
    want = hip.kv4_attention(rows, cache, pos, max_len=Lmax)
    assert torch.isfinite(want).all() and torch.equal(y[0, :n], want[0, :n]) and (want[1] == 0).all()
    for x in hip.kv4_read(cache, G._pos([0, 0]), 128):
        assert torch.isfinite(x[:, :, :Lmax]).all() and torch.isnan(x[:, :, Lmax:]).all()


def test_config_file_chooses_the_cache(hip, tmp_path):
    """config.json's kv_cache_bits holds unless load_bitnet_model is told otherwise."""
    import json

    import test_gpu_model as T
    from oracle import rotor_oracle as O
    from rotor import gpu_layers
    from rotor.bitnet_model import load_bitnet_model

    T._write_checkpoint(tmp_path, O.make_bitnet_params(6, T.SMALL, 96), T.SMALL, 96)
    file = tmp_path / "config.json"
    cfg = json.loads(file.read_text())
    gpu_layers._gpu_instance = hip
    try:
        assert load_bitnet_model(str(tmp_path), use_gpu=True).kv_cache_bits == 32
        file.write_text(json.dumps(dict(cfg, kv_cache_bits=4)))
        assert load_bitnet_model(str(tmp_path), use_gpu=True).kv_cache_bits == 4
        assert load_bitnet_model(str(tmp_path), use_gpu=True, kv_cache_bits=32).kv_cache_bits == 32
        file.write_text(json.dumps(dict(cfg, kv_cache_bits=8)))
        with pytest.raises(ValueError, match="kv_cache_bits"):
            load_bitnet_model(str(tmp_path), use_gpu=True)
    finally:
        gpu_layers._gpu_instance = None


def test_model_past_65536_positions(hip):
    """A sequence that runs past the 65536 positions of the fp32 cache: the last layer's attention over it, for nine
    tokens and for one, against 64 bits over the values that the cache holds."""
    import test_gpu_model as T
    from oracle import rotor_oracle as O

    cfg = T.SMALL
    model = T._device_model(hip, O.make_bitnet_params(77, cfg, 192), dict(cfg, kv_cache_bits=4), 70000)
    H, n, hd = cfg["n_heads"], cfg["n_layers"], cfg["d_model"] // cfg["n_heads"]
    ids = np.random.default_rng(1).integers(0, cfg["vocab_size"], 65531).astype(np.int32)
    cache = None
    for at in range(0, len(ids), 512):
        _, cache = model.forward(ids[at:at + 512], past_kv_cache=cache, use_cache=True, return_logits=False)
    table = model._dev.rope.cpu().numpy().reshape(-1, hd // 2, 2)
    for M in (9, 1):
        model._dev.trace = {}
        _, cache = model.forward(ids[:M], past_kv_cache=cache, use_cache=True)
        trace, model._dev.trace = model._dev.trace, None
        q = model._dev._state(M)["q"].cpu().numpy().reshape(1, M, H, hd)
        if M == 1:  # (rotated in the attention's launch and not kept)
            q = K4.rope(q, table, np.array([[cache.length - 1]]))
            got = trace["steps"][0]["attn"][n - 1].cpu().numpy()
        else:
            got = trace["attn"][n - 1].cpu().numpy()
        c = cache[n - 1]
        want = K4.attention(q, c["k"], c["v"], [cache.length - M])
        # (fp32 sums of 65540 numbers of random signs: below 2^-24 sqrt(2 x 65540) = 2.2e-5 of the result's own order)
        assert np.linalg.norm(got.reshape(want.shape) - want) <= 2.2e-5 * np.linalg.norm(want)
    assert cache.length == 65541
