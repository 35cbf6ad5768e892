"""The expert layer for few tokens against its definition in 64 bits."""
import math

import pytest
import torch

from onnxruntime_genai_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer(T, E, H, I, kind, bias, seed=0):
    """Arguments of the call, and the experts' numbers in 64 bits with the gate and up rows of every expert stacked."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)
    order = lambda t: ops.interleave_experts_gate_up(t, fused_interleaved=False)
    p = dict(x=n(T, H), router_w=n(E, H) / math.sqrt(H), router_b=n(E) if bias else None)
    gu_b, d_b = (n(E, 2 * I), n(E, H)) if bias else (None, None)
    if kind == "bf16":
        gu, d = n(E, 2 * I, H) / math.sqrt(H), n(E, H, I) / math.sqrt(I)
        p.update(gate_up_w=order(gu), down_w=d)
    else:
        def packed(N, K, rows):
            codes = torch.randint(0, 16, (E, N, K), dtype=torch.uint8, generator=g)
            sc = torch.randint(117, 122, (E, N, K // 32), dtype=torch.uint8, generator=g)
            if kind == "fp4 bf16 form":
                sc[0, 0, 0] = 90          # below the fp16 form's range
            half = kind != "fp4 bf16 form"
            v = ops.Fp4Experts.from_codes(codes, sc, "cpu", half=half).dequantize().to(DEV)
            return ops.Fp4Experts.from_codes(rows(codes), rows(sc), DEV, half=half), v
        (p["gate_up_w"], gu), (p["down_w"], d) = packed(2 * I, H, order), packed(H, I, lambda t: t)
    p.update(gate_up_b=order(gu_b) if bias else None, down_b=d_b)
    return p, dict(gate_up=gu, gate_up_b=gu_b, down=d, down_b=d_b)


def exact(p, w, top, weights, act, alpha, limit):
    """The layer in 64 bits, and how far the call may be off: relative steps of 2^-8 for what it rounds to 16 bits (the activations between the products, the
    result; packed experts in fp16 form: 2^-11, covered by that), fp32 sums of n products 2^-24 n of the sum of magnitudes."""
    x = p["x"].double()
    T, H = x.shape
    I = w["down"].shape[2]
    logits = x @ p["router_w"].double().T + (p["router_b"].double() if p["router_b"] is not None else 0)
    out, tol = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        vals, ids = torch.sort(logits[t], descending=True, stable=True)
        share = torch.softmax(logits[t], -1)[ids[:top]] if weights == "all" else torch.softmax(vals[:top], -1)
        for s, e in zip(share, ids[:top].tolist()):
            m = w["gate_up"][e].double()
            gu, size = m @ x[t], m.abs() @ x[t].abs()
            if w["gate_up_b"] is not None:
                gu, size = gu + w["gate_up_b"][e].double(), size + w["gate_up_b"][e].double().abs()
            g, u, dg, du = gu[:I], gu[I:], H * 2.0 ** -24 * size[:I], H * 2.0 ** -24 * size[I:]
            if act == "clamped":
                if limit > 0:
                    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
                sg = torch.sigmoid(alpha * g)
                h, dh = g * sg * (u + 1), (1 + alpha * g.abs()) * dg * (u + 1).abs() + g.abs() * du
            else:
                sg = torch.sigmoid(g)
                h, dh = g * sg * u, 1.1 * dg * u.abs() + g.abs() * du
            dh = dh + 2.0 ** -8 * h.abs() + 2.0 ** -20 * h.abs()
            d = w["down"][e].double()
            y, dy = d @ h, d.abs() @ dh + I * 2.0 ** -24 * (d.abs() @ h.abs())
            if w["down_b"] is not None:
                y = y + w["down_b"][e].double()
            out[t] += s * y
            tol[t] += s * dy + 2.0 ** -18 * s * y.abs()          # routing weight: logits in fp32, an exponential
    return out, tol + 2.0 ** -8 * out.abs() + 1e-6


KINDS = ["bf16", "fp4", "fp4 bf16 form"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E,top,H,I,weights,act", [
    (1, 8, 2, 64, 64, "selected", "silu"), (1, 32, 4, 2880, 2880, "selected", "clamped"), (2, 128, 8, 2048, 768, "renormed", "silu"),
    (8, 8, 2, 512, 1024, "selected", "silu"), (5, 60, 4, 320, 192, "all", "silu"), (8, 4, 4, 128, 448, "renormed", "clamped"),
    (7, 32, 4, 704, 576, "selected", "clamped"), (3, 1, 1, 192, 64, "all", "silu"), (8, 300, 32, 64, 64, "selected", "silu")])
def test_layer(T, E, top, H, I, weights, act, kind):
    p, w = layer(T, E, H, I, kind, act == "clamped")
    args = dict(top=top, weights=weights, act=act, alpha=1.702 if act == "clamped" else 1.0, limit=1.5 if act == "clamped" else 0.0)
    got = ops.moe_few_tokens(**p, **args)
    want, tol = exact(p, w, **args)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} times what the roundings allow"
    for t in range(T):                  # a token's result does not go by its neighbours
        alone = ops.moe_few_tokens(**{**p, "x": p["x"][t:t + 1]}, **args)
        assert bool(((alone.double() - want[t:t + 1]).abs() <= tol[t:t + 1]).all())
    assert torch.equal(ops.moe_few_tokens(**p, **args), got)


def test_columns_that_are_no_whole_vectors():
    p, w = layer(4, 8, 72, 128, "bf16", False)
    args = dict(top=2, weights="selected", act="silu", alpha=1.0, limit=0.0)
    want, tol = exact(p, w, **args)
    wide = torch.zeros(4, 99, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:75] = p["x"]
    for x in (p["x"], wide[:, 3:75], p["x"].t().contiguous().t()):
        assert bool(((ops.moe_few_tokens(**{**p, "x": x}, **args).double() - want).abs() <= tol).all())


def test_all_tokens_at_one_expert_and_equal_logits():
    p, w = layer(8, 16, 256, 128, "bf16", False)
    p["router_w"] = torch.zeros_like(p["router_w"])
    args = dict(top=3, weights="selected", act="silu", alpha=1.0, limit=0.0)
    want, tol = exact(p, w, **args)
    p["gate_up_w"][3:] = math.nan                     # experts beyond the first three are not looked at
    p["down_w"][3:] = math.nan
    assert bool(((ops.moe_few_tokens(**p, **args).double() - want).abs() <= tol).all())


def test_rows_that_are_not_numbers_stay_to_themselves():
    p, _ = layer(6, 8, 128, 64, "bf16", True)
    args = dict(top=2, weights="renormed", act="silu")
    ref = ops.moe_few_tokens(**p, **args)
    p["x"] = p["x"].clone()
    p["x"][2, 5], p["x"][4, 0] = math.nan, math.inf
    got = ops.moe_few_tokens(**p, **args)
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], ref[keep]) and bool(torch.isnan(got[2]).all())


def test_two_graphs_at_once():
    p, _ = layer(4, 32, 512, 256, "fp4", True)
    args = dict(top=4, act="clamped", alpha=1.702, limit=7.0)
    first = ops.moe_few_tokens(**p, **args)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with ops.graph_capture(g):
            y = ops.moe_few_tokens(**p, **args)
        graphs.append((g, y, torch.cuda.Stream()))
    for _ in range(3):
        for g, _, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, first) for _, y, _ in graphs)


def test_refusals_of_device_tensors():
    p, _ = layer(2, 8, 64, 64, "bf16", True)
    for kw in (dict(x=p["x"].float()), dict(router_w=p["router_w"].float()), dict(down_b=p["down_b"].float()), dict(gate_up_w=p["gate_up_w"].transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError, match="bfloat16"):
            ops.moe_few_tokens(**{**p, **kw}, top=2)
    with pytest.raises(ValueError, match="different devices"):
        ops.moe_few_tokens(**{**p, "router_b": p["router_b"].cpu()}, top=2)


def test_experts_beyond_32_bits():
    """2.4 G numbers of gate and up weights; the experts behind that border are the ones that are met."""
    T, E, top, H, I = 3, 256, 2, 4608, 1024
    g = torch.Generator(DEV).manual_seed(2)
    n = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    gate_up, down = n(E, 2 * I, H).mul_(H ** -0.5), n(E, H, I).mul_(I ** -0.5)
    p = dict(x=n(T, H), router_w=torch.zeros(E, H, dtype=torch.bfloat16, device=DEV), router_b=torch.zeros(E, dtype=torch.bfloat16, device=DEV), gate_up_b=None, down_b=None)
    p["router_b"][250:] = torch.arange(6).to(torch.bfloat16).to(DEV)
    args = dict(top=top, weights="selected", act="silu", alpha=1.0, limit=0.0)
    got = ops.moe_few_tokens(gate_up_w=gate_up, down_w=down, **p, **args)
    last = slice(250, 256)
    stacked = gate_up[last].view(6, I // 64, 2, 64, H).transpose(1, 2).reshape(6, 2 * I, H)
    want, tol = exact({**p, "router_w": p["router_w"][last], "router_b": p["router_b"][last]}, dict(gate_up=stacked, gate_up_b=None, down=down[last], down_b=None), **args)
    assert bool(((got.double() - want).abs() <= tol).all())
    ops.check_kernel_status()


@pytest.mark.parametrize("kind", KINDS)
def test_many_turns_of_the_rings_repeat(kind):
    """Stages of both rings are handed back and written again some hundred times a call, beside copies of another stream: always the same result, near the exact one."""
    T, E, H, I = 8, 4, 1024, 4096
    p, w = layer(T, E, H, I, kind, False)
    args = dict(top=2, weights="selected", act="silu", alpha=1.0, limit=0.0)
    first = ops.moe_few_tokens(**p, **args)
    want, tol = exact(p, w, **args)
    assert bool(((first.double() - want).abs() <= tol).all())
    traffic, side = torch.empty(1 << 27, dtype=torch.uint8, device=DEV), torch.cuda.Stream()
    differs = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(300):
        if i % 10 == 0:
            with torch.cuda.stream(side):
                traffic[: 1 << 26].copy_(traffic[1 << 26:])
        differs += (ops.moe_few_tokens(**p, **args) != first).any()
    torch.cuda.synchronize()
    assert int(differs) == 0
    ops.check_kernel_status()


def fixed_choice(p, E):
    """The router replaced by logits that do not go by the rows."""
    p["router_w"] = torch.zeros_like(p["router_w"])
    p["router_b"] = (torch.arange(E) % 5).to(torch.bfloat16).to(DEV)
    return p


def below(p, w, act):
    """What the activations' 16 bits may lose below the normal numbers of fp16: with the largest of 64 neighbours at 2^14 or more, half a step of 2^-24 is 2^-39 of it."""
    a = p["x"].double().abs()
    most = torch.zeros(a.shape[0], 1, dtype=torch.float64, device=DEV)
    for e in range(w["down"].shape[0]):
        g, u = (a @ w["gate_up"][e].double().abs().T).chunk(2, dim=1)
        most = torch.maximum(most, (g * (u + (act == "clamped"))).amax(1, keepdim=True) * w["down"][e].double().abs().sum(1).max())
    return 2.0 ** -39 * most


@pytest.mark.parametrize("act,limit", [("silu", 0.0), ("clamped", 1.5), ("clamped", 0.0)])
@pytest.mark.parametrize("size", [-14, -8, 0, 8])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_any_size(kind, size, act, limit):
    """Activations far below and above the range of 16-bit floats: every error is relative to what is added up, whatever its size."""
    T, E, H, I = 5, 8, 1024, 320
    p, w = layer(T, E, H, I, kind, False, seed=size + 20)
    fixed_choice(p, E)
    p["x"] = p["x"] * 2.0 ** size
    p["x"][1] *= 2.0 ** -6                             # not all tokens of one size
    args = dict(top=3, weights="selected", act=act, alpha=1.702 if act == "clamped" else 1.0, limit=limit)
    got = ops.moe_few_tokens(**p, **args).double()
    want, tol = exact(p, w, **args)
    tol = tol - 1e-6 + below(p, w, act)
    worst = float(((got - want).abs() / tol).max())
    assert worst <= 1, f"off by {worst:.3g} times what the roundings allow"
    assert float((got - want).norm() / want.norm()) < 2.0 ** -7          # (and as a whole: half a step of bf16 twice)
    ops.check_kernel_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["silu", "clamped"])
def test_infinities_are_not_cut_off(kind, act):
    p, _ = layer(6, 8, 256, 128, kind, False)
    fixed_choice(p, 8)
    args = dict(top=2, weights="renormed", act=act, alpha=1.702 if act == "clamped" else 1.0, limit=0.0)
    ref = ops.moe_few_tokens(**p, **args)
    p["x"] = p["x"].clone()
    p["x"][2, 5], p["x"][4, 0] = math.nan, math.inf
    got = ops.moe_few_tokens(**p, **args)
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], ref[keep]) and bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[4]).any())


@pytest.mark.parametrize("weights", ["selected", "all"])
def test_masked_experts(weights):
    """Router biases of minus infinity: such experts are the last to be chosen, and count nothing."""
    p, w = layer(3, 16, 128, 64, "bf16", True)
    p["router_b"][3:] = -math.inf
    args = dict(top=5, weights=weights, act="silu", alpha=1.0, limit=0.0)
    want, tol = exact(p, w, **args)
    assert bool(((ops.moe_few_tokens(**p, **args).double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_whose_logits_are_no_numbers(kind):
    """All logits of a token, or some, are NaN: the choice is short of experts.  Such a token's result is NaN every time, the others' as without it."""
    p, _ = layer(8, 16, 256, 1024, kind, False)
    args = dict(top=4, weights="selected", act="silu")
    ref = ops.moe_few_tokens(**p, **args)
    p["x"] = p["x"].clone()
    p["x"][1], p["x"][6] = math.nan, math.nan
    for _ in range(50):
        junk = torch.ones(1 << 22, dtype=torch.bfloat16, device=DEV)        # what the call's scratch may find in its memory are numbers
        del junk
        got = ops.moe_few_tokens(**p, **args)
        keep = [0, 2, 3, 4, 5, 7]
        assert torch.equal(got[keep], ref[keep]) and bool(torch.isnan(got[[1, 6]]).all())
    p["x"] = torch.where(torch.isnan(p["x"]), torch.ones_like(p["x"]), p["x"])
    fixed_choice(p, 16)
    p["router_b"][2:] = math.nan                       # two experts are left to choose four from
    assert bool(torch.isnan(ops.moe_few_tokens(**p, **args)).all())
