"""What is measured of the microscaled 4-bit products and of the expert layer for few tokens.

Three operators, each in its plain form (torch, 32 bits) and through the framework:
  quantise  rows to 4-bit floating point in blocks (NVFP4, MXFP4) and back
  linear    quantised rows times quantised weights, with bias, residual, or the gated activation of an MLP
  moe       a mixture-of-experts layer from the tokens to the weighted sum: router, choice, both products of every chosen expert
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"nvfp4": 16, "mxfp4": 32}
ROW_TOP = 6.0 * 448.0          # largest value of a row over its scale: e2m1's times e4m3's


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the rows in front of a projection of a decode step, read back as bf16: launch latency
        dict(name="quantise 8 x 4096", op="quantise", form="nvfp4", T=8, K=4096, fp32=False),
        # the rows in front of the down projection of a prompt: bandwidth
        dict(name="quantise 4096 x 14336", op="quantise", form="nvfp4", T=4096, K=14336, fp32=False),
        # rows of a 32-bit residual stream, a ragged prompt, power-of-two scales
        dict(name="quantise 777 x 2880 mxfp4", op="quantise", form="mxfp4", T=777, K=2880, fp32=True),
        # the q, k, v projection of one decoding request
        dict(name="qkv, 1 token", op="linear", form="nvfp4", T=1, K=4096, N=6144, bias=False, residual=False, pair=False),
        # the gate and up projections of a small batch
        dict(name="gate/up, 16 tokens", op="linear", form="nvfp4", T=16, K=4096, N=28672, bias=False, residual=False, pair=True),
        # the down projection of a served batch, added to the residual stream
        dict(name="down + residual, 64 tokens", op="linear", form="nvfp4", T=64, K=14336, N=4096, bias=False, residual=True, pair=False),
        # a projection with a bias over a prompt of odd length
        dict(name="777 tokens, bias, mxfp4", op="linear", form="mxfp4", T=777, K=2880, N=5120, bias=True, residual=False, pair=False),
        # the gate and up projections of a long prompt: the tensor cores
        dict(name="gate/up, 8192 tokens", op="linear", form="nvfp4", T=8192, K=4096, N=28672, bias=False, residual=False, pair=True),
        # one decoding request: packed 4-bit experts with biases and the clamped activation
        dict(name="moe 4 of 32, 1 token, mxfp4", op="moe", weights="mxfp4", rule="selected", act="clamped", T=1, E=32, top=4, H=2880, I=2880, bias=True),
        # a few decoding requests, of which some share experts
        dict(name="moe 4 of 32, 7 tokens, mxfp4", op="moe", weights="mxfp4", rule="selected", act="clamped", T=7, E=32, top=4, H=2880, I=2880, bias=True),
        # one decoding request: many narrow 16-bit experts
        dict(name="moe 8 of 128, 1 token, bf16", op="moe", weights="bf16", rule="renormed", act="silu", T=1, E=128, top=8, H=2048, I=768, bias=False),
        # few wide 16-bit experts, a batch that meets nearly all of them
        dict(name="moe 2 of 8, 8 tokens, bf16", op="moe", weights="bf16", rule="selected", act="silu", T=8, E=8, top=2, H=4096, I=14336, bias=False),
    ]


def _log_uniform(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["quantise", "linear", "linear", "moe"])
    form = rng.choice(["nvfp4", "nvfp4", "mxfp4"])
    b = BLOCK[form]
    if op == "quantise":
        return dict(op=op, form=form, T=_log_uniform(rng, 1, 4096), K=_log_uniform(rng, 2 * b, 14336, b), fp32=rng.random() < 0.3)
    if op == "linear":
        pair = rng.random() < 0.3
        N = _log_uniform(rng, 128, 28672, 128) if pair else _log_uniform(rng, 64, 28672)
        extra = not pair and rng.random() < 0.5
        return dict(op=op, form=form, T=_log_uniform(rng, 1, 8192), K=_log_uniform(rng, 4 * b, 14336, b) if N < 8192 else _log_uniform(rng, 4 * b, 4096, b),
                    N=N, bias=extra, residual=not pair and rng.random() < 0.5, pair=pair)
    weights = rng.choice(["bf16", "mxfp4"])
    E = rng.choice([8, 16, 32, 60, 64, 128])
    most = 1 << 29                                       # weights of all experts together: a part of the largest listed case's
    H = _log_uniform(rng, 256, 4096, 64)
    top_i = max(128, min(8192, most // (E * 3 * H)))
    act = rng.choice(["silu", "clamped"])
    return dict(op=op, weights=weights, rule=rng.choice(["selected", "all", "renormed"]), act=act, T=rng.randint(1, 8), E=E,
                top=rng.randint(1, min(8, E)), H=H, I=_log_uniform(rng, 128, top_i, 64), bias=act == "clamped")


# ------------------------------------------------------------------------------------------ inputs
def _codes_of(v):
    """e2m1 codes of values that are already over their scale: nearest, ties to the even code, at most 6."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return c + 8 * ((v < 0) & (c > 0)).to(torch.uint8)


def _encode(w, form):
    """A weight as a checkpoint holds it: codes two to a byte (the even column in the low half), block scales as bytes, one scale of the whole."""
    shape, b = w.shape, BLOCK[form]
    blocks = w.view(*shape[:-1], shape[-1] // b, b)
    top = blocks.abs().amax(-1)
    if form == "nvfp4":
        whole = (w.abs().amax() / ROW_TOP).reshape(1)
        sc = (top / (6.0 * whole)).to(torch.float8_e4m3fn)
        over, sc = sc.float() * whole, sc.view(torch.uint8)
    else:
        whole, e = None, torch.frexp(top)[1] - 3
        over, sc = torch.ldexp(torch.ones_like(top), e), (e + 127).to(torch.uint8)
    c = _codes_of(blocks / over[..., None].clamp(min=1e-30)).view(shape)
    return c[..., 0::2] | (c[..., 1::2] << 4), sc, whole


def _rows(T, K, g, dtype):
    """Rows as they come out of a norm: a few columns are much larger than the rest."""
    wide = torch.exp(0.7 * torch.randn(K, generator=g, device="cuda"))
    return (torch.randn(T, K, generator=g, device="cuda") * wide).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")
    st = {"case": case}
    if case["op"] == "quantise":
        st["x"] = _rows(case["T"], case["K"], g, torch.float32 if case["fp32"] else torch.bfloat16)
        return st
    if case["op"] == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        st["x"] = _rows(T, K, g, torch.bfloat16)
        st["codes"], st["scales"], st["whole"] = _encode(normal(N, K) / math.sqrt(K), case["form"])
        st["bias"] = normal(N).to(torch.bfloat16) if case["bias"] else None
        st["residual"] = normal(T, N).to(torch.bfloat16) if case["residual"] else None
        if own:
            from onnxruntime_genai_b200 import ops
            order = ops.interleave_gate_up if case["pair"] else lambda t: t
            st["w"] = ops.Fp4Matrix.from_codes(order(st["codes"]), order(st["scales"]), st["whole"], form=case["form"], interleaved=case["pair"])
        return st
    T, E, H, I = case["T"], case["E"], case["H"], case["I"]
    st["x"] = _rows(T, H, g, torch.bfloat16)
    st["router"] = (normal(E, H) / math.sqrt(H)).to(torch.bfloat16)
    st["router_b"] = normal(E).to(torch.bfloat16) if case["bias"] else None
    # [gate; up] rows of every expert
    gate_up, down = normal(E, 2 * I, H) / math.sqrt(H), normal(E, H, I) / math.sqrt(I)
    st["gate_up_b"] = (0.1 * normal(E, 2 * I)).to(torch.bfloat16) if case["bias"] else None
    st["down_b"] = (0.1 * normal(E, H)).to(torch.bfloat16) if case["bias"] else None
    if case["weights"] == "mxfp4":
        st["gate_up"], st["down"] = _encode(gate_up, "mxfp4")[:2], _encode(down, "mxfp4")[:2]
    else:
        st["gate_up"], st["down"] = gate_up.to(torch.bfloat16), down.to(torch.bfloat16)
    del gate_up, down
    if own:
        from onnxruntime_genai_b200 import ops
        order = lambda t: ops.interleave_experts_gate_up(t, fused_interleaved=False)
        if case["weights"] == "mxfp4":
            split = lambda c: torch.stack([c & 0xF, c >> 4], dim=-1).flatten(-2)
            pack = lambda c, s: ops.Fp4Experts.from_codes(split(c), s, "cuda", keep_host=False)
            st["w"] = pack(*map(order, st["gate_up"])), pack(*st["down"])
        else:
            st["w"] = order(st["gate_up"]), st["down"]
        st["w_b"] = order(st["gate_up_b"]) if case["bias"] else None
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _quantised(x, form):
    """Rows as the values that their 4-bit form stands for, in 32 bits."""
    x = x.float()
    blocks = x.view(x.shape[0], -1, BLOCK[form])
    top = blocks.abs().amax(-1)
    if form == "nvfp4":
        # the row's scale: the smallest power of two that brings its largest value under ROW_TOP (1.3125 * 2^11), so that the steps below divide exactly
        m, e = torch.frexp(top.amax(-1, keepdim=True))
        e = torch.where(m <= 1.3125 / 2, e - 12, e - 11).clamp(min=-100)
        sc = (torch.ldexp(top, -e) / torch.full_like(top, 6.0)).to(torch.float8_e4m3fn).float()
        over = torch.ldexp(sc, e)
        c = _codes_of(torch.where(sc[..., None] > 0, blocks / over[..., None], 0.0))
    else:
        e = (torch.frexp(top)[1] - 3).clamp(min=-127)
        over = torch.ldexp(torch.ones_like(top), e)
        c = _codes_of(torch.ldexp(blocks, -e[..., None]))
    return (_value(c) * over[..., None]).view(x.shape)


def _value(c):
    """The numbers of e2m1 codes 0..15."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=c.device)
    return table[c.int()]


def _decoded(codes, scales, whole, form):
    """A checkpoint's weight in 32 bits."""
    v = _value(torch.stack([codes & 0xF, codes >> 4], dim=-1).flatten(-2))
    sc = scales.view(torch.float8_e4m3fn).float() * whole if form == "nvfp4" else torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (v.view(*sc.shape, BLOCK[form]) * sc[..., None]).view(v.shape)


def _choose(logits, top, rule):
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids, best = order.indices[:, :top], order.values[:, :top]
    if rule == "all":
        return ids, torch.exp(best - logits.amax(-1, keepdim=True)) / torch.exp(logits - logits.amax(-1, keepdim=True)).sum(-1, keepdim=True)
    p = torch.exp(best - best[:, :1])
    return ids, p / p.sum(-1, keepdim=True)


def _gated(g, u, act):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    g, u = g.clamp(max=7.0), u.clamp(min=-7.0, max=7.0)
    return g / (1 + torch.exp(-1.702 * g)) * (u + 1)


def run(st):
    case, x = st["case"], st["x"]
    if own:
        from onnxruntime_genai_b200 import ops
        if case["op"] == "quantise":
            return ops.quantize_fp4(x, case["form"]).dequantize(torch.bfloat16)
        if case["op"] == "linear":
            return ops.gate_up_act(x, st["w"]) if case["pair"] else ops.linear(x, st["w"], st["bias"], st["residual"])
        return ops.moe_few_tokens(x, st["router"], st["router_b"], st["w"][0], st["w_b"], st["w"][1], st["down_b"], top=case["top"], weights=case["rule"],
                                  act=case["act"], alpha=1.702, limit=7.0 if case["act"] == "clamped" else 0.0)
    if case["op"] == "quantise":
        return _quantised(x, case["form"]).to(torch.bfloat16)
    if case["op"] == "linear":
        y = _quantised(x, case["form"]) @ _decoded(st["codes"], st["scales"], st["whole"], case["form"]).T
        if case["pair"]:
            y = _gated(*y.chunk(2, dim=1), "silu")
        if st["bias"] is not None:
            y = y + st["bias"].float()
        if st["residual"] is not None:
            y = y + st["residual"].float()
        return y.to(torch.bfloat16)
    logits = x.float() @ st["router"].float().T
    if case["bias"]:
        logits = logits + st["router_b"].float()
    ids, share = _choose(logits, case["top"], case["rule"])
    if case["weights"] == "mxfp4":
        gate_up, down = (_decoded(c[ids], s[ids], None, "mxfp4") for c, s in (st["gate_up"], st["down"]))
    else:
        gate_up, down = st["gate_up"][ids].float(), st["down"][ids].float()
    gu = (gate_up @ x.float()[:, None, :, None])[..., 0]
    if case["bias"]:
        gu = gu + st["gate_up_b"].float()[ids]
    y = (down @ _gated(*gu.chunk(2, dim=-1), case["act"])[..., None])[..., 0]
    if case["bias"]:
        y = y + st["down_b"].float()[ids]
    return (y * share[..., None]).sum(1).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "quantise":
        n = case["T"] * case["K"]
        return {"bytes": n * ((4 if case["fp32"] else 2) + 2), "flops": 2 * n}
    if case["op"] == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        out = T * (N // 2 if case["pair"] else N) * 2
        per = 0.5 + 1.0 / BLOCK[case["form"]]
        return {"bytes": int(T * K * 2 + N * K * per + out * (2 if case["residual"] else 1) + (2 * N if case["bias"] else 0)), "flops": 2 * T * N * K}
    T, E, H, I = case["T"], case["E"], case["H"], case["I"]
    met = E * (1 - (1 - case["top"] / E) ** T)          # experts that T tokens meet, on average
    per = 2.0 if case["weights"] == "bf16" else 0.5 + 1.0 / 32
    return {"bytes": int(met * 3 * H * I * per + E * H * 2 + T * H * 4), "flops": 2 * T * case["top"] * 3 * H * I + 2 * T * E * H}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _nearest64(v, mantissa, lowest, most):
    """v >= 0 rounded to a binary floating-point grid of so many stored bits, whose smallest normal number is 2^lowest."""
    e = (torch.frexp(v).exponent - 1).clamp(min=lowest)
    step = torch.ldexp(torch.ones_like(v), e - mantissa)
    return (torch.round(v / step) * step).clamp(max=most)


def _quantised64(x, form):
    T, K = x.shape
    b = x.double().reshape(T, K // BLOCK[form], BLOCK[form])
    top = b.abs().max(-1, keepdim=True).values
    if form == "nvfp4":
        most = top.max(1, keepdim=True).values
        row = torch.ldexp(torch.ones_like(most), torch.frexp(most).exponent - 12)
        row = torch.where(row * ROW_TOP < most, 2 * row, row)
        scale = _nearest64(top / (6 * row), 3, -6, 448.0) * row
    else:
        scale = torch.ldexp(torch.ones_like(top), torch.frexp(top).exponent - 3)
    return torch.where(scale > 0, torch.sign(b) * _nearest64(b.abs() / scale, 1, 0, 6.0) * scale, 0.0).reshape(T, K)


def _decoded64(codes, scales, whole, form):
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int16, device=codes.device)
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    m, e, s = c % 2, c // 2 % 4, 1 - 2 * (c // 8)
    v = (s * torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))).double()
    if form == "nvfp4":
        n = scales.to(torch.int16)
        f, x = n % 8, n // 8 % 16
        sc = torch.where(x == 0, f / 8 * 2.0 ** -6, (1 + f.double() / 8) * torch.exp2(x.double() - 7)) * whole.double()
    else:
        sc = torch.exp2(scales.double() - 127)
    return v * sc.repeat_interleave(BLOCK[form], dim=-1)


def _gated64(g, u, act):
    if act == "clamped":
        g, u = torch.minimum(g, torch.full_like(g, 7.0)), torch.maximum(torch.minimum(u, torch.full_like(u, 7.0)), torch.full_like(u, -7.0)) + 1
        return g * torch.special.expit(1.702 * g) * u
    return g * torch.special.expit(g) * u


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"]
    if case["op"] == "quantise":
        return _quantised64(x, case["form"])
    if case["op"] == "linear":
        y = torch.einsum("tk,nk->tn", _quantised64(x, case["form"]), _decoded64(st["codes"], st["scales"], st["whole"], case["form"]))
        if case["pair"]:
            half = case["N"] // 2
            y = _gated64(y[:, :half], y[:, half:], "silu")
        for more in (st["bias"], st["residual"]):
            y = y if more is None else y + more.double()
        return y
    out, x = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda"), x.double()
    logits = x @ st["router"].double().T + (st["router_b"].double() if case["bias"] else 0)
    for t in range(case["T"]):
        left, shares = logits[t].clone(), {}
        for _ in range(case["top"]):
            e = int(torch.nonzero(left == left.max())[0])
            shares[e] = float(logits[t, e])
            left[e] = -math.inf
        most = float(logits[t].max())
        total = sum(math.exp(v - most) for v in (logits[t].tolist() if case["rule"] == "all" else shares.values()))
        for e, v in shares.items():
            if case["weights"] == "mxfp4":
                gate_up, down = (_decoded64(c[e], s[e], None, "mxfp4") for c, s in (st["gate_up"], st["down"]))
            else:
                gate_up, down = st["gate_up"][e].double(), st["down"][e].double()
            gu = gate_up @ x[t] + (st["gate_up_b"][e].double() if case["bias"] else 0)
            y = down @ _gated64(gu[: case["I"]], gu[case["I"]:], case["act"]) + (st["down_b"][e].double() if case["bias"] else 0)
            out[t] += math.exp(v - most) / total * y
    return out
