"""4-bit floating-point matrices without a device: layout, rounding rules, products on the CPU, refusals."""
import math

import pytest
import torch

from onnxruntime_genai_b200 import ops
from onnxruntime_genai_b200.ops import _lib, fp4_matrix

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def nearest_e2m1(v: float) -> float:
    """Nearest number of the grid, the even code of two equally near ones, 6 beyond it."""
    a = abs(v)
    i = min(range(8), key=lambda j: (abs(GRID[j] - a), j % 2))
    return math.copysign(GRID[i], v)


def nearest_e4m3(v: float) -> float:
    if v >= 448:
        return 448.0
    e = max(math.frexp(v)[1] - 1, -6) if v else -6
    return round(v / 2.0 ** (e - 3)) * 2.0 ** (e - 3)          # round(): to even


def quantised_row(row, form):
    """The definition, number by number in 64 bits."""
    row = [float(v) for v in row]
    if not all(math.isfinite(v) for v in row):
        return [math.nan] * len(row)
    out, top = [], max(abs(v) for v in row)
    if form == "nvfp4":
        e = -100
        while top > 2688 * 2.0 ** e:
            e += 1
        for b in range(0, len(row), 16):
            blk = row[b:b + 16]
            sc = nearest_e4m3(max(abs(v) for v in blk) / 2.0 ** e / 6)
            out += [nearest_e2m1(v / (sc * 2.0 ** e)) * sc * 2.0 ** e if sc else 0.0 for v in blk]
    else:
        for b in range(0, len(row), 32):
            blk = row[b:b + 32]
            m = max(abs(v) for v in blk)
            sc = 2.0 ** max(math.frexp(m)[1] - 3, -127) if m else 1.0
            out += [nearest_e2m1(v / sc) * sc for v in blk]
    return out


def rows_of(kind, T, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g)
    if kind == "wide":
        x = x * torch.exp(3 * torch.randn(T, K // 16, generator=g)).repeat_interleave(16, 1)
    elif kind == "ties":          # multiples of an eighth: halves of steps are common
        x = torch.randint(-56, 57, (T, K), generator=g) / 8.0
    elif kind == "extremes":
        x = x * 2.0 ** torch.randint(-120, 120, (T, 1), generator=g)
        x[0] = 0.0
        x[min(1, T - 1), :16] = 0.0
        x[T // 2, K // 2] = math.inf
        x[T - 1, 0] = math.nan
    return x.to(dtype)


@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,K", [(1, 32), (7, 64), (128, 256), (130, 384), (300, 2880)])
def test_layout_holds_every_code_and_scale(form, rows, K):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (rows, K // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(1, 126, (rows, K // fp4_matrix.BLOCK[form]), dtype=torch.uint8, generator=g)
    scale = torch.rand(rows, generator=g)
    m = ops.Fp4Matrix.from_codes(codes, scales, scale, form)
    c = m.codes()
    assert m.shape == (rows, K) and torch.equal(c[:, 0::2] | c[:, 1::2] << 4, codes)
    assert torch.equal(m.scales(), scales) and torch.equal(m.row_scales(), scale)
    assert m.data.numel() == _lib.lib().ogb_fp4_matrix_bytes(rows, K, fp4_matrix.FORMS[form]) == sum(fp4_matrix.sizes(rows, K, form))
    # the byte that the kernels look a code and a scale up at (row r, k)
    kb_all, padded, block, steps = -(-K // 256), -(-rows // 128) * 128, fp4_matrix.BLOCK[form], 64 // fp4_matrix.BLOCK[form]
    for r, k in ((0, 0), (rows - 1, K - 1), (rows // 2, K // 2), (rows // 3, K - 7)):
        kb, i = divmod(k, 256)
        byte = int(m.data[(kb * padded + r) * 128 + (((i // 32) ^ (r % 8)) << 4) + i % 32 // 2])
        assert (byte >> 4 if k % 2 else byte & 15) == int(c[r, k])
        b = i // block
        at = kb_all * padded * 128 + ((kb * (padded // 128) + r // 128) * steps + b // 4) * 512 + (r % 32) * 16 + r % 128 // 32 * 4 + b % 4
        assert int(m.data[at]) == int(scales[r, k // block])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "extremes"])
def test_rows_are_rounded_as_defined(kind, form, dtype):
    x = rows_of(kind, 6, 96, dtype)
    got = ops.quantize_fp4(x, form).dequantize()
    want = torch.tensor([quantised_row(r, form) for r in x.tolist()], dtype=torch.float64).float()
    assert torch.equal(torch.nan_to_num(got, nan=7e30), torch.nan_to_num(want, nan=7e30))


def test_products_on_the_cpu():
    g = torch.Generator().manual_seed(2)
    x, wv = torch.randn(5, 128, generator=g), torch.randn(256, 128, generator=g)
    for form in ("nvfp4", "mxfp4"):
        w = ops.quantize_fp4(ops.interleave_gate_up(wv), form)
        w.interleaved = True
        q = ops.quantize_fp4(x, form)
        want = q.dequantize().double() @ w.dequantize().double().T
        # fp32 sums of 128 products: at most 128 * 2^-24 of the sum of magnitudes
        tol = 128 * 2.0 ** -24 * (q.dequantize().abs() @ w.dequantize().abs().T) + 1e-30
        assert bool(((ops.linear(x, w).double() - want).abs() <= tol).all())
        assert torch.equal(ops.linear(q, w, out_fp32=True), ops.linear(x, w))
        g_, u = want.view(5, 2, 2, 64).unbind(2)
        y = (torch.nn.functional.silu(g_) * u).reshape(5, 128)
        assert torch.allclose(ops.gate_up_act(x, w).double(), y, rtol=1e-4, atol=1e-4)
        relu = (torch.relu(g_) * u).reshape(5, 128)
        assert torch.allclose(ops.gate_up_act(x, w, act="relu").double(), relu, rtol=1e-4, atol=1e-4)


def test_refusals():
    ok = ops.quantize_fp4(torch.randn(128, 64))
    with pytest.raises(ValueError, match="blocks of 16"):
        ops.quantize_fp4(torch.randn(2, 40))
    with pytest.raises(ValueError, match="blocks of 32"):
        ops.quantize_fp4(torch.randn(2, 48), "mxfp4")
    with pytest.raises(ValueError, match="form"):
        ops.quantize_fp4(torch.randn(2, 64), "int4")
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.quantize_fp4(torch.randn(2, 64).half())
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.quantize_fp4(torch.randn(64))
    with pytest.raises(ValueError, match="rows of 32"):
        ops.linear(torch.randn(2, 32), ok)
    with pytest.raises(ValueError, match="rows in mxfp4"):
        ops.linear(ops.quantize_fp4(torch.randn(2, 64), "mxfp4"), ok)
    with pytest.raises(ValueError, match="bias"):
        ops.linear(torch.randn(2, 64), ok, bias=torch.zeros(64))
    with pytest.raises(ValueError, match="residual"):
        ops.linear(torch.randn(2, 64), ok, residual=torch.zeros(3, 128))
    with pytest.raises(ValueError, match="output"):
        ops.linear(torch.randn(2, 64), ok, out=torch.zeros(2, 64))
    with pytest.raises(ValueError, match="quantised already"):
        ops.linear(ok, ok, norm_eps=1e-5)
    with pytest.raises(RuntimeError, match="reduced over ranks"):
        ops.linear(torch.randn(2, 64), ok, all_reduce=True)
    with pytest.raises(ValueError, match="read back"):
        ok.dequantize(torch.float16)
    codes = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="shape"):
        ops.Fp4Matrix.from_codes(codes, torch.zeros(4, 3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="2 scales"):
        ops.Fp4Matrix.from_codes(codes, torch.zeros(4, 4, dtype=torch.uint8), torch.ones(2))
    with pytest.raises(ValueError, match="64 \\+ 64"):
        ops.Fp4Matrix.from_codes(codes, torch.zeros(4, 4, dtype=torch.uint8), interleaved=True)
    assert ops.linear(torch.randn(0, 64), ok).shape == (0, 128)


def test_launchers_refuse_on_the_host():
    L, A, W, C = _lib.lib(), 1 << 20, 2 << 20, 3 << 20
    assert L.ogb_fp4_matrix_bytes(4, 64, 2) == -1 and L.ogb_fp4_matrix_bytes(-1, 64, 0) == -1 and L.ogb_fp4_matrix_bytes(4, 0, 0) == -1
    assert L.ogb_quantize_fp4(A, 64, 0, 4, 40, 0, W, None) == -1          # no whole blocks
    assert L.ogb_quantize_fp4(A, 64, 0, 4, 48, 1, W, None) == -1
    assert L.ogb_quantize_fp4(A, 64, 0, 4, 64, 0, W + 8, None) == -1      # alignment of the buffer
    assert L.ogb_quantize_fp4(None, 64, 0, 4, 64, 0, W, None) == -1
    assert L.ogb_quantize_fp4(A, 64, 0, 0, 64, 0, W, None) == 0           # nothing to do
    assert L.ogb_dequantize_fp4(W, 4, 64, 0, None, 64, 0, None) == -1
    linear = lambda T=4, N=128, K=64, form=0, pair=0, res=None, w=W: L.ogb_linear_fp4(A, 64, 0, W, T, w, N, K, form, C, N, 0, pair, None, res, N, 0, None, 148, None)
    assert linear(T=-1) == -1 and linear(N=0) == -1 and linear(K=40) == -1 and linear(form=2) == -1 and linear(w=W + 4) == -1
    assert linear(N=64, pair=1) == -1 and linear(pair=1, res=C) == -1 and linear(T=0) == 0


def test_block_scales_that_are_no_numbers():
    codes = torch.full((2, 32), 0x22, dtype=torch.uint8)
    for form, good, bad in (("nvfp4", 0x7e, (0x7f, 0x80, 0xb8, 0xff)), ("mxfp4", 0xfe, (0xff,))):
        scales = torch.full((2, 64 // fp4_matrix.BLOCK[form]), 0x30, dtype=torch.uint8)
        scales[1, 1] = good
        assert bool(torch.isfinite(ops.Fp4Matrix.from_codes(codes, scales, form=form).dequantize()).all())
        for b in bad:
            scales[1, 1] = b
            with pytest.raises(ValueError, match="block scale"):
                ops.Fp4Matrix.from_codes(codes, scales, form=form)
            if form == "nvfp4":
                with pytest.raises(ValueError, match="block scale"):
                    ops.Fp4Matrix.from_codes(codes, scales.view(torch.float8_e4m3fn), form=form)
