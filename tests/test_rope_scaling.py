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
