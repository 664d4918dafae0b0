"""Scalings of the rotary tables that transformers' configurations have beside the plain
ones: the factor on cos and sin that mscale and mscale_all_dim give together."""

import types

import pytest
import torch

from blockstreamer_b200 import attention


@pytest.mark.parametrize("factor", [0.5, 1.0, 4.0, 40.0])
@pytest.mark.parametrize("extra", [
    dict(mscale=1.0, mscale_all_dim=1.0), dict(mscale=0.707, mscale_all_dim=1.0), dict(mscale=1.0, mscale_all_dim=0.5),
    dict(mscale=0.707), dict(mscale_all_dim=0.707), dict(mscale=0.0, mscale_all_dim=1.0), dict(mscale=1.0, mscale_all_dim=0),
    dict(mscale=0.7, mscale_all_dim=1.0, attention_factor=1.25),
])
def test_yarn_factor_is_that_of_transformers(factor, extra):
    hf = pytest.importorskip("transformers.modeling_rope_utils")
    scaling = dict(rope_type="yarn", factor=factor, original_max_position_embeddings=4096, **extra)
    full = dict(scaling, rope_theta=10000.0)

    class Config(types.SimpleNamespace):
        def standardize_rope_params(self):
            return None

    cfg = Config(rope_theta=10000.0, rope_scaling=full, rope_parameters=full, head_dim=64, hidden_size=256,
                 num_attention_heads=4, max_position_embeddings=131072, partial_rotary_factor=1.0)
    want, factor_out = hf.ROPE_INIT_FUNCTIONS["yarn"](cfg, torch.device("cpu"))
    got, mine = attention.rotary_frequencies(64, 10000.0, scaling)
    assert mine == pytest.approx(factor_out, rel=1e-6)
    assert bool(((got - want.double()).abs() <= 2e-6 * got).all())
