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


def test_a_shared_expert_is_a_gated_feed_forward():
    """It is a part of its layer's mixture, not one of the model's: its matrices are in 4 bits like another's, and count as such."""
    from plain_sodotar import WIDE

    from fastgen_amd.engine import Model
    from fastgen_amd.kernels.linear import Matrix4, StreamedMatrix

    config = dict(WIDE, layers=[dict(l, mlp=dict(l["mlp"], shared=dict(l["mlp"]["shared"], ff=64))) for l in WIDE["layers"]])
    model = Model.random(config, 1, torch.bfloat16, "cpu", w4_group=32)
    shared = [b.ffn.shared for b in model.parts.blocks]
    assert all(isinstance(m, Matrix4) for s in shared for m in (s.w_gate_up, s.w_down))
    assert sorted(id(m) for m in model.matrices4()) == sorted(id(m) for s in shared for m in (s.w_gate_up, s.w_down))
    plain = Model.random(config, 1, torch.bfloat16, "cpu")
    assert all(isinstance(b.ffn.shared.w_down, StreamedMatrix) for b in plain.parts.blocks) and not plain.matrices4()


def test_a_step_s_memory_counts_a_shared_expert_in_4_bits(monkeypatch):
    """What its products take beside their results: the sums of a cut, and x in fp16."""
    from plain_sodotar import WIDE

    from fastgen_amd.engine import Model
    from fastgen_amd.engine.engine import step_memory_estimate
    from fastgen_amd.kernels import ops

    monkeypatch.setattr(ops, "compute_units", lambda: 256)
    config = dict(WIDE, layers=[dict(l, mlp=dict(l["mlp"], shared=dict(l["mlp"]["shared"], ff=8192))) for l in WIDE["layers"]])
    model = Model.random(config, 1, torch.bfloat16, "cpu", w4_group=32)
    most = max(m.scratch_bytes(4096) for m in model.matrices4())
    assert most >= 2 * 4096 * 8192 and step_memory_estimate(model, 4096, 1) >= most


def test_a_model_without_a_matrix_for_4_bits_is_refused():
    from plain_zudisun import ONLY_SCAN

    from fastgen_amd.engine import Model

    with pytest.raises(ValueError, match="no matrix"):
        Model.random(ONLY_SCAN, 1, torch.bfloat16, "cpu", w4_group=32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 17, 96, 130])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "relu", "limited"])
def test_a_gated_feed_forward_in_4_bits(activation, m):
    """Every activation, at the rows of every kernel, against 64 bits: the products' errors as their own tests have them, which the activation (of slopes up
    to 1.13) and the down projection hand on; 2^-18 for the activation itself, half a step of bfloat16 where its result is rounded, and one of gate and up where
    the activation is a kernel of its own behind a bfloat16 product."""
    from test_weight4 import DEV, _in_64, _to, _x

    from fastgen_amd.config import PartSpec
    from fastgen_amd.kernels.linear import Matrix4, four_bits
    from fastgen_amd.kernels.twins import w4_values
    from fastgen_amd.parts import build_part

    dim, hidden, limit, alpha = 256, 192, 1.5, 1.7
    options = dict(dim=dim, hidden_dim=hidden, activation=activation, **(dict(limit=limit, alpha=alpha) if activation == "limited" else {}))
    part = build_part("feed_forward", PartSpec("swiglu", "f", options))
    g = torch.Generator().manual_seed(m)
    with four_bits(64):
        part.load({s.name: torch.randn(s.shape, generator=g) / s.shape[1] ** 0.5 for s in part.tensor_specs()}, torch.bfloat16, DEV)
    assert isinstance(part.w_gate_up, Matrix4) and isinstance(part.w_down, Matrix4)
    x, many = _x(m, m, dim), m > 96
    own = part.separate  # (then gate and up are float32)
    y, tol = _in_64(x, _to(part.w_gate_up.w, "cpu"), rounded=many and not own, out_half=2.0**-24 if own else 2.0**-8 if activation == "gelu_tanh" else 0.0)
    (gate, up), (tg, tu) = ([h.reshape(m, hidden) for h in t.view(m, -1, 2, 8).unbind(2)] for t in (y, tol))
    if activation == "limited":
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit) + 1
        f = gate * torch.sigmoid(alpha * gate)
    else:
        f = dict(silu=torch.nn.functional.silu, relu=torch.relu, gelu_tanh=lambda v: torch.nn.functional.gelu(v, approximate="tanh"))[activation](gate)
    act = f * up
    off = 1.13 * tg * up.abs() + (f.abs() + 1.13 * tg) * tu + 2.0**-18 * (gate * up).abs()
    off = off + 2.0**-8 * (act.abs() + off)
    down = _to(part.w_down.w, "cpu")
    want, tol = _in_64(act, down, rounded=many)
    tol = 1.02 * tol + 1.01 * (off @ w4_values(down).double().abs().T)
    got = part.forward(x.to(DEV)).cpu().double()
    got = got.sum(0) if got.dim() == 3 else got
    share = float(((got - want).abs() / tol).max())
    assert got.shape == (m, dim) and share <= 1, share


@pytest.mark.gpu
def test_a_mixture_whose_shared_expert_is_in_4_bits(tmp_path):
    """The model against the plain one with the shared experts' matrices rounded the same way: a choice of experts within rounding of a tie may fall the
    other way than in the plain bfloat16 run, so nine in ten positions keep to twice what that run is off."""
    import traces
    from helpers import run_trace, save_model_folder
    from plain_sodotar import WIDE, plain_forward, plain_weights
    from test_gpu_sodotar import _close_to_plain, _tokens

    from fastgen_amd.engine import Model, ModelRunner
    from fastgen_amd.kernels.twins import w4_values
    from fastgen_amd.kernels.weight4 import quantize_w4

    config = dict(WIDE, layers=[dict(l, mlp=dict(l["mlp"], shared=dict(l["mlp"]["shared"], ff=64))) for l in WIDE["layers"]])
    weights = {k: v.to(torch.bfloat16).float() for k, v in plain_weights(config, 3).items()}
    folder = save_model_folder(tmp_path, config, weights)
    small = {k: w4_values(quantize_w4(v, 32)) if any(f"shared.{n}" in k for n in ("gate", "up", "down")) else v for k, v in weights.items()}
    assert sum(not torch.equal(small[k], weights[k]) for k in weights) == 6
    lengths = {"a": 3, "b": 20, "c": 70}
    tokens = _tokens(config, lengths, 1)
    want = {r: plain_forward(small, config, t, torch.float32) for r, t in tokens.items()}
    noise = {r: plain_forward(small, config, t, torch.bfloat16) for r, t in tokens.items()}
    model = Model.from_folder(folder, torch.bfloat16, "cuda:0", w4_group=32)
    assert len(model.matrices4()) == 4
    trace = traces.tail(lengths)
    got = run_trace(ModelRunner(model, page_size=16, max_tokens=traces.max_live_tokens(trace, round_to=64), max_requests=4), trace, tokens)
    _close_to_plain(got, want, noise, torch.bfloat16, "shared experts in 4 bits", True)


def test_arguments_that_ask_for_other_weights_than_the_model_has(model, monkeypatch):
    """A model that is there already keeps its weights: arguments that ask for others are refused; those that say nothing take it as it is."""
    from fastgen_amd.engine import Model

    from fastgen_amd.kernels import ops

    monkeypatch.setattr(ops, "compute_units", lambda: 256)
    with pytest.raises(ValueError, match="groups of 32"):
        Fastgen.from_model(model, GenArgs(w4_group=32, max_seq=256), ())
    small = Model.random(TINY, 1, torch.bfloat16, "cpu", w4_group=32)
    with pytest.raises(ValueError, match="groups of 64"):
        Fastgen.from_model(small, GenArgs(w4_group=64, max_seq=256), ())
    for args in (GenArgs(max_seq=256), GenArgs(w4_group=32, max_seq=256)):
        assert Fastgen.from_model(small, args, ()).engine.model is small
