"""The expert layer for few tokens without a device: its restatement against a plain one, refusals."""
import pytest
import torch

from onnxruntime_genai_b200 import ops
from onnxruntime_genai_b200.ops import _lib


def layer(T=3, E=8, H=64, I=64, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    return dict(x=n(T, H), router_w=n(E, H) / 8, router_b=n(E) if bias else None, gate_up_w=n(E, 2 * I, H) / 8, gate_up_b=n(E, 2 * I) / 8 if bias else None,
                down_w=n(E, H, I) / 8, down_b=n(E, H) / 8 if bias else None)


@pytest.mark.parametrize("weights", ["selected", "all", "renormed"])
@pytest.mark.parametrize("act", ["silu", "clamped"])
def test_restatement(weights, act):
    p = layer()
    got = ops.moe_few_tokens(top=2, weights=weights, act=act, alpha=1.702, limit=1.0, **p)
    d = {k: v.double() for k, v in p.items()}
    probs = torch.softmax(d["x"] @ d["router_w"].T + d["router_b"], -1)
    for t in range(3):
        w, ids = probs[t].topk(2)
        if weights != "all":
            w = w / w.sum()
        want = 0
        for s, e in zip(w, ids):
            gu = d["gate_up_w"][e] @ d["x"][t] + d["gate_up_b"][e]
            g, u = gu[:64], gu[64:]
            if act == "clamped":
                g, u = g.clamp(max=1.0), u.clamp(-1.0, 1.0)
                h = g * torch.sigmoid(1.702 * g) * (u + 1)
            else:
                h = torch.nn.functional.silu(g) * u
            want = want + s * (d["down_w"][e] @ h + d["down_b"][e])
        assert torch.allclose(got[t].double(), want, rtol=1e-4, atol=1e-5)


def test_equal_logits_go_to_the_lowest_index():
    p = layer(T=1, bias=False)
    p["router_w"][:] = 0
    a = ops.moe_few_tokens(top=2, **p)
    p["gate_up_w"][2:] = float("nan")
    assert torch.equal(ops.moe_few_tokens(top=2, **p), a)


def test_refusals():
    p = layer()
    bad = lambda **kw: {**p, **kw}
    for kw, match in ((dict(x=torch.randn(9, 64)), "1 to 8"), (dict(x=torch.randn(0, 64)), "1 to 8"), (dict(x=torch.randn(2, 32)), "do not fit"),
                      (dict(router_w=torch.randn(4, 64)), "do not fit"), (dict(down_w=torch.randn(8, 64, 32)), "do not fit"),
                      (dict(down_b=torch.randn(8, 32)), "bias"), (dict(router_b=torch.randn(3)), "bias")):
        with pytest.raises(ValueError, match=match):
            ops.moe_few_tokens(top=2, **bad(**kw))
    with pytest.raises(ValueError, match="experts"):
        ops.moe_few_tokens(top=9, **p)
    with pytest.raises(ValueError, match="experts"):
        ops.moe_few_tokens(top=0, **p)
    with pytest.raises(ValueError, match="sigmoid"):
        ops.moe_few_tokens(top=2, weights="sigmoid", **p)
    with pytest.raises(ValueError, match="relu2"):
        ops.moe_few_tokens(top=2, act="relu2", **p)
    with pytest.raises(ValueError, match="blocks of 64"):
        ops.moe_few_tokens(top=2, **layer(I=32))
    codes = torch.randint(0, 16, (8, 128, 64), dtype=torch.uint8)
    packed = ops.Fp4Experts.from_codes(codes, torch.full((8, 128, 2), 120, dtype=torch.uint8), "cpu")
    with pytest.raises(ValueError, match="one form"):
        ops.moe_few_tokens(top=2, **bad(gate_up_w=packed))


def test_launcher_refuses_on_the_host():
    L, A = _lib.lib(), 1 << 20
    assert L.ogb_moe_few_scratch_bytes(0, 2, 64) == -1 and L.ogb_moe_few_scratch_bytes(9, 2, 64) == -1 and L.ogb_moe_few_scratch_bytes(1, 33, 64) == -1
    call = lambda T=1, H=64, I=64, E=8, top=2, rule=0, weights=0, act=1: L.ogb_moe_few_tokens(A, 64, A, None, A, None, A, None, A, T, H, I, E, top, rule, weights, act, 1.0,
                                                                                              0.0, A, None, 148, None)
    assert call(T=0) == -1 and call(T=9) == -1 and call(I=32) == -1 and call(E=1) == -1 and call(E=2000) == -1 and call(rule=3) == -1
    assert call(weights=3) == -1 and call(act=0) == -1 and call(H=68, weights=1) == -1 and call(H=0) == -1
