"""Angles scaled for long contexts: what a config.json's "rope_scaling" says reaches the angles, or is refused before
anything is loaded."""
import numpy as np
import pytest

from rotor.bitnet_model import BitNetModel, config_from_hf, rope_table

HF = dict(vocab_size=64, hidden_size=512, num_hidden_layers=1, num_attention_heads=4, intermediate_size=256, max_position_embeddings=4096)
YARN = {"rope_type": "yarn", "factor": 4.0}


def test_yarn_takes_the_context_from_the_config():
    """A file that leaves original_max_position_embeddings out means its max_position_embeddings."""
    for missing in ({}, {"original_max_position_embeddings": None}):
        got = config_from_hf(dict(HF, rope_scaling={**YARN, **missing}))["rope_scaling"]
        assert got == {**YARN, "original_max_position_embeddings": 4096}
        assert np.isfinite(rope_table(100, 128, 1e4, got)).all()
    named = {**YARN, "original_max_position_embeddings": 1024}
    assert config_from_hf(dict(HF, rope_scaling=named))["rope_scaling"] == named
    linear = {"type": "linear", "factor": 2.0}
    assert config_from_hf(dict(HF, rope_scaling=linear))["rope_scaling"] == linear


def model_config(**kw):
    return dict(vocab_size=64, d_model=512, n_layers=1, n_heads=4, n_kv_heads=2, d_ff=256, max_seq_len=64, **kw)


@pytest.mark.parametrize("bad", [{"rope_type": "llama3", "factor": 8.0}, {"type": "dynamic", "factor": 2.0}, {"rope_type": "longrope"},
                                 {"rope_type": "linear", "factor": -1.0}, {"rope_type": "yarn", "factor": 2.0}, {"factor": 2.0}])
def test_refused_with_the_config(bad):
    """The constructor says so, with the config alone: no weight has been read and no device looked for."""
    with pytest.raises(ValueError, match="rope_scaling"):
        BitNetModel(model_config(rope_scaling=bad), use_gpu=True)


def amplitude(**kw):
    t = rope_table(4, 64, 1e4, {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, **kw})
    a = np.hypot(t[..., 0].astype(np.float64), t[..., 1])
    assert np.ptp(a) < 1e-6
    return a.mean()


def test_yarn_amplitude():
    """attention_factor, or the ratio of 0.1 m ln f + 1 for mscale and for mscale_all_dim, or that with 1 alone."""
    ln = np.log(40.0)
    for want, kw in ((0.1 * ln + 1, {}), (1.0, dict(mscale=1.0, mscale_all_dim=1.0)), (1.0, dict(mscale=0.707, mscale_all_dim=0.707)),
                     ((0.1 * ln + 1) / (0.05 * ln + 1), dict(mscale=1.0, mscale_all_dim=0.5)), (0.1 * ln + 1, dict(mscale=1, mscale_all_dim=0)),
                     (1.25, dict(attention_factor=1.25)), (1.25, dict(attention_factor=1.25, mscale=1.0, mscale_all_dim=0.5)),
                     (0.1 * ln + 1, dict(attention_factor=None, mscale=None, mscale_all_dim=None, truncate=None))):
        assert abs(amplitude(**kw) - want) < 1e-6, kw
    for alone in (dict(mscale=0.707), dict(mscale_all_dim=1.0)):
        with pytest.raises(ValueError, match="rope_scaling: .*mscale"):
            amplitude(**alone)


def frequencies(rotary, theta, **kw):
    """Each pair's angle at position 1, over what it is without scaling."""
    t = rope_table(2, rotary, theta, {"rope_type": "yarn", "attention_factor": 1.0, **kw})[1].astype(np.float64)
    plain = theta ** (-np.arange(0, rotary, 2) / rotary)
    return np.arctan2(t[:, 1], t[:, 0]) / plain


@pytest.mark.parametrize("truncate", [True, False])
def test_yarn_mixed_frequencies(truncate):
    """The ramp worked out by hand.  rotary 16, theta 2^16: pair i turns n 2^(-2 i) / (2 pi) times in n positions.  With n = 2^13 pi
    it is 2^(12 - 2 i): beta_fast 2^7 turns is pair 2.5, beta_slow 2 is pair 5.5."""
    got = frequencies(16, 65536.0, factor=8.0, original_max_position_embeddings=2.0 ** 13 * np.pi, beta_fast=128, beta_slow=2, truncate=truncate)
    ramp = [0, 0, 0, 1 / 4, 2 / 4, 3 / 4, 1, 1] if truncate else [0, 0, 0, 1 / 6, 3 / 6, 5 / 6, 1, 1]  # from 2 to 6, or 2.5 to 5.5
    want = np.array([1 - r + r / 8 for r in ramp])
    assert np.allclose(got, want, rtol=1e-6, atol=0)


@pytest.mark.parametrize("bad", [{"rope_type": "linear", "factor": 2.0, "attention_factor": 2.0}, {"rope_type": "linear", "factor": 2.0, "rope_theta": 5e5},
                                 {"rope_type": "ntk", "factor": 2.0, "alpha": 3.0}, {"rope_type": "ntk", "factor": 2.0, "beta_fast": 32},
                                 {**YARN, "original_max_position_embeddings": 4096, "short_factor": [1.0]},
                                 {**YARN, "original_max_position_embeddings": 4096, "high_freq_factor": 4.0}])
def test_keys_that_a_type_does_not_take(bad):
    """... and might change the angles are refused, not dropped."""
    with pytest.raises(ValueError, match="rope_scaling: .*" + list(bad)[-1]):
        rope_table(4, 64, 1e4, bad)


def test_keys_that_change_nothing():
    """Null, a type under both names, what another program noted; the context that a type does not go by; plain angles by name."""
    plain = rope_table(50, 64, 1e4)
    for kind in ("linear", "ntk"):
        want = rope_table(50, 64, 1e4, {"type": kind, "factor": 2.0})
        assert not np.array_equal(want, plain)
        assert np.array_equal(want, rope_table(50, 64, 1e4, {"rope_type": kind, "type": kind, "factor": 2, "finetuned": True, "alpha": None,
                                                             "original_max_position_embeddings": 4096}))
    assert np.array_equal(plain, rope_table(50, 64, 1e4, {"rope_type": "default", "mrope_section": [16, 8, 8]}))
    assert np.array_equal(plain, rope_table(50, 64, 1e4, {}))


@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn"])
@pytest.mark.parametrize("name,values", [
    ("factor", [0, -2.0, float("inf"), float("nan"), "two", [2.0]]), ("original_max_position_embeddings", [0, -5, float("inf"), float("nan"), "long"]),
    ("beta_fast", [0, -1, 0.5, float("nan"), "x"]), ("beta_slow", [0, -1, 33, float("inf")]), ("attention_factor", [0, -1, float("nan"), "x"]),
    ("mscale", [-1, float("nan"), "x"]), ("mscale_all_dim", [-1, float("inf")]), ("truncate", [0, "no"])])
def test_values_out_of_range(kind, name, values):
    """A ValueError that names the key, and neither a table of NaN nor another error."""
    whole = dict(rope_type=kind, factor=4.0)
    if kind == "yarn":
        whole.update(original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=1.0)
    elif name != "factor":
        return
    rope_table(4, 64, 1e4, whole)
    for v in values:
        with np.errstate(all="raise"), pytest.raises(ValueError, match="rope_scaling: .*" + name):
            rope_table(4, 64, 1e4, {**whole, name: v})


def test_a_factor_is_needed():
    for kind in ("linear", "ntk", "yarn"):
        for missing in ({}, {"factor": None}):
            with pytest.raises(ValueError, match="rope_scaling: factor"):
                rope_table(4, 64, 1e4, {"rope_type": kind, "original_max_position_embeddings": 4096, **missing})
    assert np.array_equal(rope_table(4, 64, 1e4, {"rope_type": "default", "factor": None}), rope_table(4, 64, 1e4))


def test_odd_forms():
    for bad in ("linear", ["linear", 2.0], 4):
        with pytest.raises(ValueError, match="rope_scaling"):
            rope_table(4, 64, 1e4, bad)
        with pytest.raises(ValueError, match="rope_scaling"):
            BitNetModel(model_config(rope_scaling=bad), use_gpu=True)
    for theta in (1.0, 0.5):  # (the pair that turns so often: no such number)
        with np.errstate(all="raise"), pytest.raises(ValueError, match="rope_scaling: .*theta"):
            rope_table(4, 64, theta, {**YARN, "original_max_position_embeddings": 4096})
    assert np.isfinite(rope_table(4, 64, 1.0, {"rope_type": "linear", "factor": 2.0})).all()
