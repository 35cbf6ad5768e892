"""Models whose NVFP4 weights stay packed (OGB_FP4_LINEAR=1) and whose experts take the kernels for few tokens (OGB_MOE_FEW=1), without a device."""
import copy

import numpy as np
import pytest
import torch

import onnxruntime_genai_b200 as og
from onnxruntime_genai_b200 import ops
from onnxruntime_genai_b200.models import moe
from onnxruntime_genai_b200.models.arch import ArchConfig
from onnxruntime_genai_b200.models.builder import export_model, random_state_dict
from onnxruntime_genai_b200.models.decoder import LayerWeights
from onnxruntime_genai_b200.ops import fp4_matrix

BASE = dict(vocab_size=211, hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128, context_length=256, bos_token_id=0,
            eos_token_id=210, pad_token_id=0)
KINDS = {"gated": {}, "biases": dict(attn_bias=True, o_bias=True), "gelu": dict(activation="gelu"),
         "norms over heads": dict(model_type="qwen3", qk_norm=True)}                          # separate q, k and v nodes


def logits(model, prompt, more=()):
    p = og.GeneratorParams(model)
    p.set_search_options(max_length=128, batch_size=prompt.shape[0])
    g = og.Generator(model, p)
    g.append_tokens(prompt)
    out = [g.get_logits()[:, -1, :].copy()]
    for t in more:
        g.append_tokens(t)
        out.append(g.get_logits()[:, -1, :].copy())
    return np.stack(out)


@pytest.mark.parametrize("kind", list(KINDS))
def test_packed_weights_and_their_products(kind, tmp_path, monkeypatch):
    arch = ArchConfig(**{**BASE, **KINDS[kind]})
    sd = random_state_dict(arch, seed=17, std=0.1)
    export_model(copy.deepcopy(arch), str(tmp_path), "fp32", "cpu", state_dict=sd, linear_format="nvfp4")
    expanded = og.Model(str(tmp_path))
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    packed = og.Model(str(tmp_path))
    for lw, le in zip(packed.decoder.layers, expanded.decoder.layers):
        for name in ("qkv_w", "o_w", "gate_up_w", "down_w"):
            w, e = getattr(lw, name), getattr(le, name)
            assert isinstance(w, ops.Fp4Matrix) and torch.is_tensor(e)
            rows = ops.interleave_gate_up(e) if name == "gate_up_w" and lw.gate_up_interleaved else e
            # code * block scale is exact and one rounding brings the global scale in; expanded: scale * global rounds, then times the code.  Three half
            # steps of 2^-24, and a fourth for their products
            assert bool(((w.dequantize() - rows).abs() <= 4 * 2.0 ** -24 * rows.abs()).all())
        assert lw.gate_up_interleaved == lw.gate_up_w.interleaved == (arch.activation == "silu")
    assert isinstance(packed.decoder.lm_head_w, ops.Fp4Matrix)
    prompt = np.random.RandomState(4).randint(0, 210, size=(1, 9)).astype(np.int32)
    more = [np.full((1, 1), t, dtype=np.int32) for t in (5, 77)]
    got = logits(packed, prompt, more)
    # the plain form: the expanded weights, and rows that are quantised and read back before each product
    plain_linear, plain_act = ops.linear, ops.gate_up_act
    monkeypatch.setattr(ops, "linear", lambda x, w, *a, **k: plain_linear(fp4_matrix.quantize(x, "nvfp4").dequantize(), w, *a, **k))
    monkeypatch.setattr(ops, "gate_up_act", lambda x, w, *a, **k: plain_act(fp4_matrix.quantize(x, "nvfp4").dequantize(), w, *a, **k))
    want = logits(expanded, prompt, more)
    # the same numbers meet in both; sums in another order could move a code at a tie, which moves an output by a step of 1/6 of a block's largest magnitude
    # times a weight: a few percent of the outputs' spread over 64 columns
    assert np.abs(got - want).max() < 0.1 * want.std()


def test_weights_are_expanded_unless_asked(tmp_path, monkeypatch):
    arch = ArchConfig(**BASE)
    export_model(copy.deepcopy(arch), str(tmp_path), "fp32", "cpu", state_dict=random_state_dict(arch, seed=1, std=0.1), linear_format="nvfp4")
    monkeypatch.delenv("OGB_FP4_LINEAR", raising=False)
    assert torch.is_tensor(og.Model(str(tmp_path)).decoder.layers[0].qkv_w)


def test_layers_the_few_token_form_takes(monkeypatch):
    lw = LayerWeights(None, None, None, None)
    lw.router_w, lw.exp_gate_up_w, lw.exp_down_w = (torch.zeros(s, dtype=torch.bfloat16) for s in ((8, 64), (8, 256, 64), (8, 64, 128)))
    spec = moe.MoeSpec(8, 2)
    x = torch.zeros(8, 64, dtype=torch.bfloat16)
    assert not moe._few_ok(lw, spec, x)                                  # it is asked for
    monkeypatch.setattr(moe, "_FEW", True)
    assert moe._few_ok(lw, spec, x) and moe._few_ok(lw, spec, x[:1])
    assert not moe._few_ok(lw, spec, x[:0]) and not moe._few_ok(lw, spec, torch.zeros(9, 64, dtype=torch.bfloat16)) and not moe._few_ok(lw, spec, x.float())
    for other in (dict(weights="sigmoid"), dict(weights="sparse_mixer"), dict(act="relu2")):
        assert not moe._few_ok(lw, moe.MoeSpec(8, 2, **other), x)
    wide = torch.zeros(8, 1 << 14, dtype=torch.bfloat16)
    lw.exp_gate_up_w = torch.zeros(1, 256, 1, dtype=torch.bfloat16).expand(8, 256, 1 << 14)
    assert moe._few_ok(lw, spec, wide[:1]) and not moe._few_ok(lw, spec, wide)           # eight rows of it do not fit shared memory
    lw.exp_gate_up_w = torch.zeros(8, 256, 64, dtype=torch.bfloat16)
    lw.exp_shared = True
    assert not moe._few_ok(lw, spec, x)
    lw.exp_shared, lw.shared_gate_up_w = False, torch.zeros(2, 2)
    assert not moe._few_ok(lw, spec, x)


def test_bytes_of_packed_weights(tmp_path, monkeypatch):
    arch = ArchConfig(**BASE)
    export_model(copy.deepcopy(arch), str(tmp_path), "fp32", "cpu", state_dict=random_state_dict(arch, seed=1, std=0.1), linear_format="nvfp4")
    expanded = og.Model(str(tmp_path)).decoder
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    packed = og.Model(str(tmp_path)).decoder
    pairs = [(packed.lm_head_w, expanded.lm_head_w)] + [(getattr(a, n), getattr(b, n)) for a, b in zip(packed.layers, expanded.layers) for n in ("qkv_w", "o_w", "gate_up_w", "down_w")]
    assert packed.weight_bytes() - expanded.weight_bytes() == sum(p.data.numel() - 4 * e.numel() for p, e in pairs)
