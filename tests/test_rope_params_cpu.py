"""Keys of a config's rotary scaling that q4llm.rope.rope_params has to take into account, or refuse."""

import math

import pytest
import torch

from q4llm.rope import rope_params

CFG = dict(hidden_size=512, num_attention_heads=8, head_dim=64, max_position_embeddings=4096)


def yarn(d, theta, factor, trained, fast=32, slow=1, truncate=True):
    """The frequencies in 64 bits: interpolated by `factor` from the dim of `slow` turns on, kept up to that of `fast`."""
    lo, hi = (d * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (fast, slow))
    if truncate:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, d - 1)
    out = []
    for i in range(d // 2):
        f = theta ** (-2 * i / d)
        r = min(max((i - lo) / (hi - lo), 0), 1)
        out.append(f / factor * r + f * (1 - r))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("theta", [10000.0, 500000.0])
@pytest.mark.parametrize("keys,mscale", [
    (dict(mscale=1.0, mscale_all_dim=1.0), 1.0),
    (dict(mscale=1.0, mscale_all_dim=0.5), (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)),
    (dict(mscale=0.707), 0.1 * math.log(40) + 1), (dict(mscale_all_dim=0.707), 0.1 * math.log(40) + 1),
    (dict(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.1), 1.1), (dict(truncate=False), 0.1 * math.log(40) + 1),
    (dict(truncate=False, beta_fast=20, beta_slow=2), 0.1 * math.log(40) + 1), (dict(truncate=True), 0.1 * math.log(40) + 1)])
def test_yarn_keys(keys, mscale, theta):
    got = rope_params({**CFG, "rope_theta": theta, "rope_scaling": {
        "rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 2048, **keys}})
    want = yarn(64, theta, 40.0, 2048, keys.get("beta_fast", 32), keys.get("beta_slow", 1), keys.get("truncate", True))
    # theta^x in fp32: x is off by 2^-24 of itself, its power by ln(theta) times that (13.2), then about eight roundings; a weight
    # of the ramp near 0 or 1 is off by 2^-23 of the frequency that it interpolates from, up to 40 times the result
    assert ((got.inv_freq.double() - want).abs() <= (14 + 8 + 2 * 40) * 2.0 ** -24 * want).all()
    assert abs(got.mscale - mscale) <= 1e-12


def test_dynamic_grows_from_the_config_length():
    """max_position_embeddings is the length that the base is kept to, whatever original_max_position_embeddings says."""
    for n in (100, 3000, 4096, 10000):
        plain = rope_params({**CFG, "rope_scaling": {"rope_type": "dynamic", "factor": 2.0}}, seq_len=n)
        given = rope_params({**CFG, "rope_scaling": {"rope_type": "dynamic", "factor": 2.0,
                                                     "original_max_position_embeddings": 2048}}, seq_len=n)
        assert torch.equal(plain.inv_freq, given.inv_freq)
        base = 10000.0 * (2.0 * max(n, 4096) / 4096 - 1) ** (64 / 62)
        want = base ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
        assert ((given.inv_freq.double() - want).abs() <= 32 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("scaling", [
    {"rope_type": "yarn", "factor": 4.0, "short_factor": [1.0]}, {"rope_type": "default", "mrope_section": [16, 8, 8]},
    {"rope_type": "linear", "factor": 2.0, "truncate": False}, {"rope_type": "longrope", "factor": 2.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "mscale": 2.0,
     "original_max_position_embeddings": 1024}])
def test_unknown_keys_are_refused(scaling):
    with pytest.raises(NotImplementedError):
        rope_params({**CFG, "rope_scaling": scaling})


def test_keys_without_a_value_are_none():
    """(And `finetuned`, which tells only how a model was made.)"""
    a = rope_params({**CFG, "rope_scaling": {"rope_type": "yarn", "factor": 4.0}})
    b = rope_params({**CFG, "rope_scaling": {"type": "yarn", "rope_type": "yarn", "factor": 4.0, "mscale": None, "attention_factor": None, "finetuned": True,
                                             "short_factor": None}})
    assert torch.equal(a.inv_freq, b.inv_freq) and a.mscale == b.mscale


@pytest.mark.parametrize("scaling", [
    {"rope_type": "yarn", "factor": 40.0, "mscale": 1.0, "mscale_all_dim": 0.5, "original_max_position_embeddings": 2048},
    {"rope_type": "yarn", "factor": 40.0, "mscale": 0.707}, {"rope_type": "yarn", "factor": 32.0, "truncate": False},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}])
def test_the_same_as_transformers(scaling):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    got = rope_params({**CFG, "rope_theta": 10000.0, "rope_scaling": dict(scaling)}, seq_len=10000)
    try:
        c = LlamaConfig(**CFG, rope_theta=10000.0, rope_parameters={**scaling, "rope_theta": 10000.0})
        want, factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](c, "cpu", seq_len=10000)
    except (KeyError, TypeError, AttributeError):
        pytest.skip("another form of this library's configs")
    assert ((got.inv_freq - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all() and abs(got.mscale - factor) <= 1e-6
