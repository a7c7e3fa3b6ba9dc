"""Layers that differ, over a cache of 8 bits and with weights in 4: windows whose pages go back, an entry that reads another one's cache, attention sinks, output
gates, values that are keys, and no rotation, through the engine against the plain model with the same numbers rounded the same way."""

import pytest
import torch

import test_gpu_parts as parts
import traces
from helpers import assert_close, run_trace
from plain_llama import plain_rmsnorm, plain_swiglu
from test_gpu_low_bits import _rounded_kv, _weights_in_4_bits
from test_gpu_parts import _hybrid_case, _HybridArch, _plain_hybrid, hybrid_arch  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LENGTHS = {"a": 150, "b": 33, "c": 5, "d": 97}


def _tokens(vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return {r: torch.randint(0, vocab, (n,), generator=g).tolist() for r, n in LENGTHS.items()}


def _compare(model, want, noise, what):
    from fastgen_amd.engine import ModelRunner

    # (so few pages that those which a window gives back are another request's next)
    runner = ModelRunner(model, page_size=32, max_tokens=416, max_requests=4, kv_dtype="e4m3")
    tokens = _tokens(211, 4)
    for tr in (traces.whole(LENGTHS), traces.tail(LENGTHS), traces.chunks(LENGTHS), traces.mixed(LENGTHS, max_live=2, seed=2)):
        assert_close(run_trace(runner, tr, tokens), want, torch.bfloat16, noise, what)
    assert all(runner.cache.free_pages(g) == 13 for g in range(len(runner.groups)))
    return runner


@pytest.mark.parametrize("w4", [0, 32])
def test_windows_and_an_entry_that_reads_another_one_s_cache(tmp_path, hybrid_arch, monkeypatch, w4):  # noqa: F811
    from fastgen_amd.engine import Model

    args = dict(dim=96, vocab=211, eps=2e-6, theta=5000.0, layers=[
        dict(mixer="attention", H=4, KV=2, hd=32, F=160),
        dict(mixer="attention", H=3, KV=1, hd=64, rot=16, window=40, F=96),
        dict(mixer="attention", H=8, KV=2, hd=32, F=224),
    ], order=[(0, None), (1, None), (1, None), (2, 0)])
    folder, w = _hybrid_case(tmp_path, args)
    if w4:
        w = _weights_in_4_bits(w, w4)
    attend = parts.plain_attention
    monkeypatch.setattr(parts, "plain_attention", lambda q, k, v, window=None: attend(q, _rounded_kv(k), _rounded_kv(v), window))
    tokens = _tokens(211, 4)
    want, noise = ({r: _plain_hybrid(w, args, t, {}, dtype) for r, t in tokens.items()} for dtype in (torch.float32, torch.bfloat16))
    runner = _compare(Model.from_folder(folder, torch.bfloat16, DEV, w4_group=w4), want, noise, f"windows, groups of {w4}")
    assert sorted(g.need.window or 0 for g in runner.groups) == [0, 40]


class _Options(_HybridArch):
    """Two layers: sinks and an output gate behind a rotation, then values that are the keys, without one, gated too."""

    name = "OptionsTestModel"

    def layout(self, a):
        out = super().layout(a)
        for layer, l in zip(out.layers, a["layers"]):
            layer.mixer.options.update(l["more"])
        return out


def _plain_options(w, a, tokens, dtype):
    from plain_llama import plain_rope_frequencies, plain_rope_interleaved, plain_rope_shuffle

    T, w = len(tokens), {k: v.to(dtype) for k, v in w.items()}
    h = w["emb.weight"][torch.tensor(tokens)]
    seen = torch.ones(T, T, dtype=torch.bool).tril()
    for i, l in enumerate(a["layers"]):
        p, H, KV, hd = f"blocks.{i}", l["H"], l["KV"], l["hd"]
        x = plain_rmsnorm(h, w[f"{p}.n1.weight"], a["eps"])
        q, k = ((x @ w[f"{p}.attn.{n}_proj.weight"].T).view(T, heads, hd) for n, heads in (("q", H), ("k", KV)))
        v = k if l["more"].get("value_from_key") else (x @ w[f"{p}.attn.v_proj.weight"].T).view(T, KV, hd)
        if l.get("pos", "rope") == "rope":
            f = plain_rope_frequencies(hd, a["theta"])
            turned = []
            for t, heads in ((q, H), (k, KV)):
                perm = plain_rope_shuffle(torch.eye(heads * hd, dtype=dtype), heads)
                turned.append(plain_rope_interleaved((t.reshape(T, heads * hd) @ perm.T).view(T, heads, hd), torch.arange(T), f))
            q, k = turned
        k, v = _rounded_kv(k), _rounded_kv(v)
        out = []
        for j in range(H):
            s = (q[:, j].float() @ k[:, j * KV // H].float().T * hd**-0.5).masked_fill(~seen, float("-inf"))
            sink = w[f"{p}.attn.sinks"][j].float().expand(T, 1) if l["more"].get("sink") else torch.full((T, 1), float("-inf"))
            out.append(torch.softmax(torch.cat([s, sink], 1), 1)[:, :T] @ v[:, j * KV // H].float())
        out = torch.cat(out, 1).to(dtype)
        out = (out.float() * torch.sigmoid((x @ w[f"{p}.attn.gate_proj.weight"].T).float())).to(dtype)
        h = h + out @ w[f"{p}.attn.o_proj.weight"].T
        x = plain_rmsnorm(h, w[f"{p}.n2.weight"], a["eps"])
        h = h + plain_swiglu(x, *(w[f"{p}.ffn.{n}_proj.weight"] for n in ("gate", "up", "down")))
    return (plain_rmsnorm(h, w["final.weight"], a["eps"]) @ w["head.weight"].T).float()


@pytest.mark.parametrize("w4", [0, 32])
def test_sinks_gates_and_values_that_are_keys(tmp_path, w4):
    from safetensors.torch import load_file, save_file

    from fastgen_amd.config import register_architecture, unregister_architecture
    from fastgen_amd.engine import Model
    from fastgen_amd.weights import write_model_folder

    args = dict(dim=96, vocab=211, eps=2e-6, theta=5000.0, order=[(0, None), (1, None)], layers=[
        dict(mixer="attention", H=4, KV=2, hd=32, F=160, more=dict(sink=True, output_gate=True)),
        dict(mixer="attention", H=6, KV=1, hd=64, F=96, pos="none", more=dict(value_from_key=True, output_gate=True))])
    register_architecture(_Options(), replace=True)
    try:
        folder = write_model_folder(tmp_path, dict(args, architectures=["OptionsTestModel"]), seed=5)
        w = load_file(str(folder / "model.safetensors"))
        # (sharp scores in the first layer; the second's keys are its values)
        w = {k: (v * 6 if "0.attn.q_proj" in k or "0.attn.k_proj" in k else v).to(torch.bfloat16).float() for k, v in w.items()}
        save_file(w, str(folder / "model.safetensors"))
        model = Model.from_folder(folder, torch.bfloat16, DEV, w4_group=w4)
        if w4:  # (the output gate's rows are part of a layer's first matrix)
            w = _weights_in_4_bits(w, w4)
        tokens = _tokens(211, 4)
        want, noise = ({r: _plain_options(w, args, t, dtype) for r, t in tokens.items()} for dtype in (torch.float32, torch.bfloat16))
        _compare(model, want, noise, f"options, groups of {w4}")
    finally:
        unregister_architecture("OptionsTestModel")
