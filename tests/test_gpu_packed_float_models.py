"""4-bit products and the expert layer for few tokens together: as calls of one step, and inside models."""
import copy

import numpy as np
import pytest
import torch

import onnxruntime_genai_b200 as og
from onnxruntime_genai_b200 import ops
from onnxruntime_genai_b200.models import moe
from onnxruntime_genai_b200.models.arch import ArchConfig
from onnxruntime_genai_b200.models.builder import export_model, random_state_dict
from test_gpu_fp4_matrix import close, weight
from test_gpu_moe_few import exact, layer
from test_packed_float_models import logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T,H,I,form,kind", [(1, 2880, 1024, "mxfp4", "fp4"), (3, 512, 768, "nvfp4", "bf16"), (8, 1024, 2048, "nvfp4", "fp4 bf16 form")])
def test_a_step_of_all_of_them(T, H, I, form, kind):
    """Rows quantised once for two products, a gated product and the one behind it with the stream as its residual, and an expert layer on the sum: run
    eagerly, captured, and replayed with other rows; every stage against its definition from the tensors that it was given."""
    p, e = layer(T, 16, H, 256, kind, False, seed=T)
    args = dict(top=4, weights="selected", act="silu", alpha=1.0, limit=0.0)
    side_w, gate_up, down = weight(640, H, form, 1), weight(2 * I, H, form, 2, interleaved=True), weight(H, I, form, 3)
    x = p.pop("x")

    def step():
        q = ops.quantize_fp4(x, form)
        a = ops.linear(q, side_w)
        h = ops.gate_up_act(q, gate_up)
        y = ops.linear(h, down, residual=x)
        return q, a, h, y, ops.moe_few_tokens(y, **p, **args)

    def check(q, a, h, y, z):
        xq, wq = q.dequantize().double(), side_w.dequantize().double()
        close(a, xq @ wq.T, xq.abs() @ wq.abs().T, H)
        wq = gate_up.dequantize().double()
        g, u = (v.reshape(T, I) for v in (xq @ wq.T).view(T, I // 64, 2, 64).unbind(2))
        sg, su = (v.reshape(T, I) for v in (xq.abs() @ wq.abs().T).view(T, I // 64, 2, 64).unbind(2))
        want, d = torch.nn.functional.silu(g) * u, (H / 16 + 8) * 2.0 ** -23
        assert bool(((h.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs() + d * (1.1 * sg * (u.abs() + d * su) + g.abs() * su) + 1e-30).all())
        hq, wq = ops.quantize_fp4(h, form).dequantize().double(), down.dequantize().double()
        close(y, hq @ wq.T + x.double(), hq.abs() @ wq.abs().T + x.double().abs(), I)
        want, tol = exact({**p, "x": y}, e, **args)
        assert bool(((z.double() - want).abs() <= tol).all())

    first = step()
    check(*first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with ops.graph_capture(g, stream=side):
        captured = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(s, f) for s, f in zip(captured[1:], first[1:]))
    x.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(91)).to(torch.bfloat16))
    g.replay()
    torch.cuda.synchronize()
    check(*captured)
    ops.check_kernel_status()


def exact_product(x, w, bias, residual, out_fp32, pair):
    """What a 4-bit product stands for, in 64 bits, and how far it may be off: the bounds of `close` (and of a gated product: silu's slope is at most 1.1)."""
    q, m = (x if isinstance(x, ops.Fp4Matrix) else ops.quantize_fp4(x, w.form)).dequantize().double(), w.dequantize().double()
    y, size, d = q @ m.T, q.abs() @ m.abs().T, (w.K / 16 + 8) * 2.0 ** -23
    for t in (bias, residual):
        if t is not None:
            y, size = y + t.double(), size + t.double().abs()
    tol = d * size
    if pair:
        (g, u), (sg, su) = ((v.reshape(len(y), -1) for v in t.view(len(y), -1, 2, 64).unbind(2)) for t in (y, size))
        y = torch.nn.functional.silu(g) * u
        tol = d * (1.1 * sg * (u.abs() + d * su) + g.abs() * su) + 2.0 ** -20 * y.abs()
    return y, tol + (0.0 if out_fp32 else 2.0 ** -8) * y.abs() + 1e-30


def exact_experts(x, router_w, router_b, gate_up_w, gate_up_b, down_w, down_b, top, weights, act, alpha, limit):
    experts = lambda w: torch.stack([w.dequantize(i).to(x.device) for i in range(w.shape[0])]) if isinstance(w, ops.Fp4Experts) else w
    stacked = lambda t: None if t is None else t.view(t.shape[0], -1, 2, 64, *t.shape[2:]).transpose(1, 2).reshape(t.shape)
    return exact(dict(x=x, router_w=router_w, router_b=router_b), dict(gate_up=stacked(experts(gate_up_w)), gate_up_b=stacked(gate_up_b), down=experts(down_w),
                 down_b=down_b), top, weights, act, alpha, limit)


def generated(model, prompt, steps):
    p = og.GeneratorParams(model)
    p.set_search_options(max_length=prompt.shape[1] + steps, batch_size=prompt.shape[0])
    g = og.Generator(model, p)
    g.append_tokens(prompt)
    seen = []
    for _ in range(steps):
        g.generate_next_token()
        seen.append(g.get_logits().copy())
    return np.stack(seen)


def checked(model, prompt, more, monkeypatch):
    """Runs a prompt and the steps behind it with every product and expert layer on the way held against its definition on the same rows."""
    calls = {"product": 0, "experts": 0}
    product, experts = ops._linear_fp4, ops.moe_few_tokens

    def near(got, want, tol, name):
        calls[name] += 1
        worst = float(((got.double() - want).abs() / tol).max())
        assert worst <= 1, f"{name} {calls[name]}: off by {worst:.3g} times what the roundings allow"
        return got

    def products(x, w, bias=None, residual=None, out_fp32=False, out=None, pair=False):
        want = exact_product(x, w, bias, residual, out_fp32, pair)
        return near(product(x, w, bias, residual, out_fp32, out, pair), *want, "product")
    with monkeypatch.context() as m:
        m.setenv("OGB_GENERATOR_GRAPH", "0")
        m.setattr(ops, "_linear_fp4", products)
        m.setattr(ops, "moe_few_tokens", lambda *a: near(experts(*a), *exact_experts(*a), "experts"))
        logits(model, prompt, more)
    ops.check_kernel_status()
    return calls


@pytest.mark.parametrize("bias", [False, True])
def test_model_with_packed_projections(bias, tmp_path, monkeypatch):
    arch = ArchConfig(vocab_size=1000, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64, intermediate_size=512, context_length=256,
                      bos_token_id=0, eos_token_id=999, pad_token_id=0, attn_bias=bias, o_bias=bias)
    d = str(tmp_path)
    export_model(copy.deepcopy(arch), d, "bf16", "cuda", state_dict=random_state_dict(arch, seed=5, std=0.05), linear_format="nvfp4")
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    model = og.Model(d)
    lw = model.decoder.layers[0]
    assert all(isinstance(w, ops.Fp4Matrix) and w.is_cuda for w in (lw.qkv_w, lw.o_w, lw.gate_up_w, lw.down_w, model.decoder.lm_head_w))
    for tokens in (7, 100):                         # a prompt's products: those for few tokens, and those on pairs of SMs
        prompt = np.random.RandomState(tokens).randint(0, 999, size=(1, tokens)).astype(np.int32)
        calls = checked(model, prompt, [np.full((1, 1), t, dtype=np.int32) for t in (5, 77, 123)], monkeypatch)
        assert calls["product"] == 9 * 4
    prompt = np.random.RandomState(1).randint(0, 999, size=(3, 11)).astype(np.int32)
    replayed = generated(model, prompt, 8)                      # from graphs, three sequences a step
    monkeypatch.setenv("OGB_GENERATOR_GRAPH", "0")
    assert np.array_equal(replayed, generated(model, prompt, 8))


@pytest.mark.parametrize("precision", ["int4", "bf16"])
def test_model_with_experts_for_few_tokens(precision, tmp_path, monkeypatch):
    """Packed projections beside experts (MXFP4 or bf16) that take the kernels for few tokens: prompts of up to eight tokens and every step after them."""
    arch = ArchConfig(vocab_size=1024, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=4, head_dim=64, intermediate_size=128, context_length=256,
                      bos_token_id=0, eos_token_id=1023, pad_token_id=0, model_type="gptoss", num_experts=8, experts_per_token=2, attn_bias=True, o_bias=True,
                      mlp_bias=True, attn_sinks=True, sliding_window=16, sliding_layers=[0])
    d = str(tmp_path)
    export_model(copy.deepcopy(arch), d, precision, "cuda", state_dict=random_state_dict(arch, seed=4, std=0.05), linear_format="nvfp4")
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    model = og.Model(d)
    lw = model.decoder.layers[0]
    assert isinstance(lw.qkv_w, ops.Fp4Matrix) and isinstance(lw.exp_gate_up_w, ops.Fp4Experts) == (precision == "int4")
    more = [np.full((1, 1), t, dtype=np.int32) for t in (5, 77, 123)]
    prompt = np.random.RandomState(6).randint(0, 1023, size=(1, 8)).astype(np.int32)
    monkeypatch.setattr(moe, "_FEW", True)
    calls = checked(model, prompt, more, monkeypatch)
    assert calls["experts"] == 2 * 4 and calls["product"] == 5 * 4
    nine = np.random.RandomState(7).randint(0, 1023, size=(1, 9)).astype(np.int32)
    with monkeypatch.context() as m:
        m.setattr(ops, "moe_few_tokens", None)      # more tokens: not called
        logits(model, nine)
    prompt = np.random.RandomState(1).randint(0, 1023, size=(4, 11)).astype(np.int32)
    replayed = generated(model, prompt, 8)                      # from graphs, four sequences a step
    monkeypatch.setenv("OGB_GENERATOR_GRAPH", "0")
    assert np.array_equal(replayed, generated(model, prompt, 8))


def test_engine_with_packed_weights_and_experts(tmp_path, monkeypatch):
    """Requests of different lengths in one engine: steps of prompts, of a few tokens and of padded batches."""
    arch = ArchConfig(vocab_size=1024, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=4, head_dim=64, intermediate_size=128, context_length=256,
                      bos_token_id=0, eos_token_id=1023, pad_token_id=0, model_type="gptoss", num_experts=8, experts_per_token=2, attn_bias=True, o_bias=True,
                      mlp_bias=True, attn_sinks=True, sliding_window=16, sliding_layers=[0])
    d = str(tmp_path)
    export_model(copy.deepcopy(arch), d, "int4", "cuda", state_dict=random_state_dict(arch, seed=8, std=0.05), linear_format="nvfp4", paged=True, block_size=16,
                 num_blocks=256, max_batch_size=16)
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    monkeypatch.setattr(moe, "_FEW", True)
    model = og.Model(d)
    engine = og.Engine(model)
    rng = np.random.RandomState(3)
    requests = []
    for n in (5, 70, 1, 9, 33):
        gp = og.GeneratorParams(model)
        gp.set_search_options(max_length=n + 12)
        r = og.Request(gp)
        r.add_tokens(rng.randint(1, 1000, size=n).astype(np.int32))
        engine.add_request(r)
        requests.append(r)
    seen = {id(r): [] for r in requests}
    while engine.has_pending_requests():
        r = engine.step()
        if r is not None:
            while r.has_unseen_tokens():
                seen[id(r)].append(r.get_unseen_token())
    ops.check_kernel_status()
    assert all(0 < len(t) <= 12 and all(0 <= v < 1024 for v in t) for t in seen.values())


def run_engine(engine, model, lengths, new):
    rng = np.random.RandomState(3)
    requests = []
    for n in lengths:
        gp = og.GeneratorParams(model)
        gp.set_search_options(max_length=n + new, min_length=n + new)
        r = og.Request(gp)
        r.add_tokens(rng.randint(1, 1000, size=n).astype(np.int32))
        engine.add_request(r)
        requests.append(r)
    seen = {id(r): [] for r in requests}
    while engine.has_pending_requests():
        r = engine.step()
        if r is not None:
            while r.has_unseen_tokens():
                seen[id(r)].append(r.get_unseen_token())
    ops.check_kernel_status()
    return [seen[id(r)] for r in requests]


@pytest.mark.parametrize("few", [False, True])
def test_every_call_of_an_engine(few, tmp_path, monkeypatch):
    """Prompts, mixed steps and padded batches of an engine: every product and expert layer against its definition on the rows it was given (padded rows may hold anything,
    and are looked at only where they are numbers); and batches that need no padding give the same tokens from graphs as eagerly."""
    from onnxruntime_genai_b200.engine.engine import ModelExecutor
    arch = ArchConfig(vocab_size=1024, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=4, head_dim=64, intermediate_size=128, context_length=256,
                      bos_token_id=0, eos_token_id=1023, pad_token_id=0, model_type="gptoss", num_experts=8, experts_per_token=2, attn_bias=True, o_bias=True,
                      mlp_bias=True, attn_sinks=True, sliding_window=16, sliding_layers=[0])
    d = str(tmp_path)
    export_model(copy.deepcopy(arch), d, "int4", "cuda", state_dict=random_state_dict(arch, seed=8, std=0.05), linear_format="nvfp4", paged=True, block_size=16,
                 num_blocks=256, max_batch_size=16)
    monkeypatch.setenv("OGB_FP4_LINEAR", "1")
    monkeypatch.setenv("OGB_ENGINE_RUN_AHEAD", "0")
    monkeypatch.setenv("OGB_ENGINE_LOOKAHEAD", "0")
    monkeypatch.setattr(moe, "_FEW", few)
    model = og.Model(d)
    lengths = (5, 70, 1, 9, 33, 2, 17, 8)
    replayed = run_engine(og.Engine(model), model, lengths, 12)
    assert all(len(t) == 12 for t in replayed)

    def eager(self, bb, cb):
        s = self._step_inputs(bb, bb, self.staging.table_cols, 1, cb * self.kv.block_size, ordered=self.order_attention)
        logits = torch.empty(bb, 1024, dtype=torch.float32, device=DEV)
        return type("Step", (), {"replay": lambda _: logits.copy_(self.decoder.forward(s, self.kv))})(), logits

    calls = {"product": 0, "experts": 0}
    product, experts = ops._linear_fp4, ops.moe_few_tokens

    def near(got, want, tol, name):
        calls[name] += 1
        rows = torch.isfinite(want).all(-1)
        assert bool(((got.double() - want).abs() <= tol)[rows].all()) and not bool(torch.isfinite(got[~rows].double()).all(-1).any()), f"{name} {calls[name]}"
        return got

    def products(x, w, bias=None, residual=None, out_fp32=False, out=None, pair=False):
        want = exact_product(x, w, bias, residual, out_fp32, pair)
        return near(product(x, w, bias, residual, out_fp32, out, pair), *want, "product")
    monkeypatch.setattr(ModelExecutor, "_capture", eager)
    assert run_engine(og.Engine(model), model, lengths, 12) == replayed
    monkeypatch.setattr(ops, "_linear_fp4", products)
    monkeypatch.setattr(ops, "moe_few_tokens", lambda *a: near(experts(*a), *exact_experts(*a), "experts"))
    run_engine(og.Engine(model), model, lengths[:5], 6)                      # steps of one token a request are padded to eight
    assert calls["product"] >= 5 * 6 and (calls["experts"] >= 2 * 5) == few
