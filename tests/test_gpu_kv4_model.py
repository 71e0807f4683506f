"""BitNetModel with the KV cache in 4 bits (kv_cache_bits=4): everything but the attention is held to the
oracle bit for bit, step by step, continuing from the device's attention outputs; the attention itself to
its 64-bit form over the values that the cache gives back."""
import numpy as np
import pytest

import test_gpu_model as T
from oracle import kv4_oracle as K4
from oracle import rotor_oracle as O

pytestmark = pytest.mark.gpu

CFGS = {"hd64": T.SMALL, "hd128": T.HD128}


@pytest.fixture(scope="module")
def models(hip):
    out = {}
    for name, cfg in CFGS.items():
        params = O.make_bitnet_params(31 + len(name), cfg, 192)
        out[name] = (T._device_model(hip, params, dict(cfg, kv_cache_bits=4), 192), params, cfg)
    return out


@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("graph", [True, False])
def test_greedy_matches_oracle(models, name, graph):
    """The prompt and every step: the oracle, continuing from the device's attention outputs and tokens, has the same
    hidden state bit for bit and logits within the head's tolerance; every token is the argmax of its logits."""
    model, params, cfg = models[name]
    prompt = np.random.default_rng(5).integers(0, cfg["vocab_size"], 130).astype(np.int32)
    model._dev.trace = {}
    try:
        toks = model.generate_greedy(prompt, 8, graph=graph)
    finally:
        trace, model._dev.trace = model._dev.trace, None
    recs = [(prompt, trace["prefill"], [a.cpu().numpy() for a in trace["attn"]])]
    recs += [(toks[i:i + 1], st, [a[None] for a in st["attn"].cpu().numpy()]) for i, st in enumerate(trace["steps"])]
    assert len(recs) == 8
    oc, E32 = {}, T._embed32(params)
    for i, (ids, rec, attn) in enumerate(recs):
        xo = []
        hn, lg64 = O.bitnet_forward(params, cfg, np.asarray(ids, np.int32), oc, attn_in=attn, x_out=xo)
        lg = rec["logits"].cpu().numpy()
        assert np.array_equal(rec["h"].cpu().numpy(), xo[0][-1]), f"hidden state of step {i}"
        T.check_logits(lg, lg64, E32, hn[-1], f"step {i}")
        assert toks[i] == int(np.argmax(lg))


@pytest.mark.parametrize("name", list(CFGS))
def test_attention_and_cache(models, name):
    """After a prompt and after single steps: the last layer's attention output is its definition over the values
    that the cache handle gives, and these are within a step of the keys and values of the oracle."""
    model, params, cfg = models[name]
    ids = np.random.default_rng(9).integers(0, cfg["vocab_size"], 70).astype(np.int32)
    H, Hkv, n = cfg["n_heads"], cfg["n_kv_heads"], cfg["n_layers"]
    hd = cfg["d_model"] // H
    model._dev.trace = {}
    try:
        _, cache = model.forward(ids, use_cache=True)
        trace = model._dev.trace
        oc = {}
        O.bitnet_forward(params, cfg, ids, oc, attn_in=[a.cpu().numpy() for a in trace["attn"]])
        rows = [(len(ids), trace["attn"][n - 1].cpu().numpy())]
        for step in range(3):
            model._dev.trace = {}
            _, cache = model.forward(np.array([step + 5], np.int32), past_kv_cache=cache, use_cache=True)
            rows.append((1, model._dev.trace["steps"][0]["attn"][n - 1].cpu().numpy()[None]))
            M, got = rows[-1] if step else rows[0]
            if step == 0:  # the prompt's rows: its queries are still in the state of its length
                q = model._dev._state(M)["q"].cpu().numpy().reshape(1, M, H, hd)
                c = cache[n - 1]
                want = K4.attention(q, c["k"], c["v"], [0])
                assert np.linalg.norm(got.reshape(want.shape) - want) <= 2e-6 * np.linalg.norm(want)
            M, got = rows[-1]
            # (one token's queries are rotated in the attention's launch and not kept)
            table = model._dev.rope.cpu().numpy().reshape(-1, hd // 2, 2)
            q = K4.rope(model._dev._state(1)["q"].cpu().numpy().reshape(H, hd), table, cache.length - 1)[None, None]
            c = cache[n - 1]
            assert c["k"].shape == c["v"].shape == (1, Hkv, cache.length, hd)
            want = K4.attention(q, c["k"], c["v"], [cache.length - 1])
            assert np.linalg.norm(got.reshape(want.shape) - want) <= 2e-6 * np.linalg.norm(want)
    finally:
        model._dev.trace = None
    for li in range(n):
        c = cache[li]
        for x, key in ((c["k"][0, :, :len(ids)], "k"), (c["v"][0, :, :len(ids)], "v")):
            ref = np.asarray(oc[li][key], np.float32).reshape(Hkv, -1, hd)[:, :len(ids)]
            _, z, h = K4.quantise(ref)
            # (the definition's own error: half a step, h; codes next to a border may fall either way, since the
            # oracle's RoPE rounds each product)
            bound = np.repeat(h * (1 + 16 * 2.0 ** -8) + np.abs(z) * 2.0 ** -7, 64, -1) + 1e-5
            assert (np.abs(x - ref) <= bound).all()


def test_forward_equals_generate(models):
    """forward's steps (one token a call, a captured graph) and generate_greedy's give the same tokens."""
    model, params, cfg = models["hd128"]
    prompt = np.random.default_rng(3).integers(0, cfg["vocab_size"], 40).astype(np.int32)
    toks = model.generate_greedy(prompt, 6)
    logits, cache = model.forward(prompt, use_cache=True)
    got = [int(np.argmax(logits[-1]))]
    for _ in range(5):
        logits, cache = model.forward(np.array(got[-1:], np.int32), past_kv_cache=cache, use_cache=True)
        got.append(int(np.argmax(logits[0])))
    # (the prompt's last logits come from the head over all rows in forward, another order of sums)
    assert got[0] == toks[0] and list(toks) == got


def test_long_cache_of_small_model(hip):
    """More positions than the fp32 cache takes (65536): a prompt near the end of 70000."""
    cfg = T.SMALL
    params = O.make_bitnet_params(77, cfg, 192)
    model = T._device_model(hip, params, dict(cfg, kv_cache_bits=4), 70000)
    ids = np.random.default_rng(1).integers(0, cfg["vocab_size"], 30).astype(np.int32)
    _, cache = model.forward(ids, use_cache=True)
    _, cache = model.forward(ids[:9], past_kv_cache=cache, use_cache=True)
    lg, cache = model.forward(ids[:1], past_kv_cache=cache, use_cache=True)
    assert cache.length == 40 and np.isfinite(lg).all() and np.isfinite(cache[0]["k"]).all()


def test_refusals(hip):
    params = O.make_bitnet_params(1, T.SMALL, 64)
    with pytest.raises(ValueError, match="kv_cache_bits"):
        T._device_model(hip, params, dict(T.SMALL, kv_cache_bits=8), 64)
    narrow = dict(T.SMALL, n_heads=T.SMALL["d_model"] // 32, n_kv_heads=T.SMALL["d_model"] // 64, kv_cache_bits=4)
    with pytest.raises(ValueError, match="head_dim"):
        T._device_model(hip, params, narrow, 64)
    with pytest.raises(ValueError, match="max_seq_len"):
        T._device_model(hip, params, dict(T.SMALL, kv_cache_bits=4), (1 << 20) + 1)


def test_load_bitnet_model_takes_the_bits(hip, tmp_path):
    import json

    from rotor import gpu_layers
    from rotor.bitnet_model import load_bitnet_model

    cfg = T.SMALL
    params = O.make_bitnet_params(6, cfg, 96)
    T._write_checkpoint(tmp_path, params, cfg, 96)
    assert json.loads((tmp_path / "config.json").read_text())["hidden_size"] == cfg["d_model"]
    gpu_layers._gpu_instance = hip
    try:
        small, full = (load_bitnet_model(str(tmp_path), use_gpu=True, kv_cache_bits=b) for b in (4, 32))
    finally:
        gpu_layers._gpu_instance = None
    ids = np.arange(20, dtype=np.int32)
    a, ca = small.forward(ids, use_cache=True)
    b, cb = full.forward(ids, use_cache=True)
    assert a.shape == b.shape and np.isfinite(a).all()
    # the first layer's keys and values see no attention before them: the same but for the 4 bits
    for key in ("k", "v"):
        x, y = ca[0][key], cb[0][key]
        _, z, h = K4.quantise(y)
        assert (np.abs(x - y) <= np.repeat(h * (1 + 16 * 2.0 ** -8) + np.abs(z) * 2.0 ** -7, 64, -1) + 1e-5).all()
