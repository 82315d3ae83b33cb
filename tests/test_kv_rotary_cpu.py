"""The rotary table's scaling: what a model's configuration may hold there is
either applied or refused."""
import pytest
import torch

from test_speed_scalesweep_b200 import kv_cache

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 64}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}


def table(scaling, base=10000.0):
    return kv_cache.rotary_cos_sin_cache(9, 16, base=base, scaling=scaling, device="cpu")


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 4.0}, LLAMA3, YARN])
def test_the_base_comes_from_one_place(scaling):
    plain = dict(scaling or {})
    assert torch.equal(table(dict(plain, rope_theta=500000.0), 500000.0), table(scaling, 500000.0))
    assert torch.equal(table(dict(plain, rope_theta=None, partial_rotary_factor=0.5)), table(scaling))
    with pytest.raises(ValueError, match="rope_theta"):
        table(dict(plain, rope_theta=500000.0))


@pytest.mark.parametrize("scaling,needle", [
    (dict(YARN, attn_factor=0.5), "attn_factor"), (dict(YARN, extrapolation_factor=0.5), "extrapolation_factor"),
    ({"rope_type": "linear", "factor": 2.0, "attention_factor": 2.0}, "attention_factor"),
    ({"rope_type": "default", "factor": 2.0}, "factor"), ({"factor": 2.0}, "factor"),
    (dict(LLAMA3, alpha=3.0), "alpha"), ({"rope_type": "linear"}, "needs factor"),
    ({k: v for k, v in YARN.items() if k != "original_max_position_embeddings"}, "needs original"),
    (dict(LLAMA3, low_freq_factor=None), "needs low_freq_factor")])
def test_what_is_not_applied_is_refused(scaling, needle):
    with pytest.raises(ValueError, match=needle):
        table(scaling)


def test_absent_and_default_keys():
    assert torch.equal(table(dict(YARN, beta_fast=None, beta_slow=1.0, truncate=True, mscale=None)), table(YARN))
    assert torch.equal(table({"type": "linear", "factor": 4.0}), table({"rope_type": "linear", "factor": 4.0}))
    assert torch.equal(table({"rope_type": "default", "mrope_section": [2, 3, 3]}), table(None))
