"""The options of a cache in 8 bits and of weights in 4, as they are written down for users (CPU: nothing is run)."""

import pytest
import torch

from plain_llama import TINY_B

from fastgen_amd.generate import Fastgen, GenArgs

E4M3 = torch.float8_e4m3fn
# heads of 32, widths that groups of 32 divide
TINY = dict(TINY_B, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, intermediate_size=256, num_hidden_layers=2)


@pytest.fixture(scope="module")
def model():
    from fastgen_amd.engine import Model

    return Model.random(TINY, 1, torch.bfloat16, "cpu")


NAMES = [("e4m3", E4M3), (E4M3, E4M3), ("model", torch.bfloat16), (None, torch.bfloat16), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.parametrize("given,held", NAMES)
def test_the_cache_by_its_name(model, given, held):
    from fastgen_amd.engine import Engine, ModelRunner

    runner = ModelRunner(model, max_tokens=256, kv_dtype=given)
    assert runner.kv_dtype == held and runner.storage.k[0].dtype == held and (runner.storage.scales[0] is not None) == (held == E4M3)
    assert Engine(model, max_tokens=256, max_batch=2, kv_dtype=given).runner.storage.k[0].dtype == held
    assert Engine.from_config(TINY, 1, device="cpu", max_tokens=256, max_batch=2, kv_dtype=given).runner.kv_dtype == held


@pytest.mark.parametrize("given,held", NAMES)
def test_generation_arguments_by_the_cache_s_name(model, given, held):
    """Also where the cache's tokens follow from a budget: half the bytes a token but for its scales."""
    # a page of 64 tokens, 2 layers, keys and values, 2 heads of 32 in 2 bytes: 32,768
    args = GenArgs(kv_dtype=given, gpu_gb=(model.weight_bytes() + 10 * 32768) / 1e9, prefill_gb=0, max_batch=2)
    runner = Fastgen.from_model(model, args, ()).engine.runner
    assert runner.storage.k[0].dtype == held
    assert runner.storage.k[0].shape[1] == (20 if held == E4M3 else 10)
    assert Fastgen.from_model(model, GenArgs(kv_dtype=given, max_seq=256, max_batch=2), ()).engine.runner.kv_dtype == held


@pytest.mark.parametrize("given", ["fp8", "E4M3", "", torch.float16, torch.float32, torch.float8_e5m2])
def test_other_caches_are_refused(model, given):
    from fastgen_amd.engine import ModelRunner

    with pytest.raises(ValueError, match="cache"):
        ModelRunner(model, max_tokens=256, kv_dtype=given)
    with pytest.raises(ValueError, match="cache"):
        Fastgen.from_model(model, GenArgs(kv_dtype=given, gpu_gb=1.0, prefill_gb=0), ())
