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
