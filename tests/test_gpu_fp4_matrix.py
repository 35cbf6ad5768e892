"""4-bit floating-point rows and products against their definition in 64 bits."""
import math

import pytest
import torch

from onnxruntime_genai_b200 import ops
from onnxruntime_genai_b200.ops import fp4_matrix
from test_fp4_matrix import rows_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weight(N, K, form, seed=3, interleaved=False):
    g = torch.Generator().manual_seed(seed)
    w = fp4_matrix.quantize(torch.randn(N, K, generator=g) / math.sqrt(K), form)
    c = w.codes()
    return ops.Fp4Matrix.from_codes(c[:, 0::2] | c[:, 1::2] << 4, w.scales(), w.row_scales(), form, DEV, interleaved)


def close(y, want, size, K):
    """A product within its rounding to bf16 (half a step, 2^-8 of the value) and its fp32 sums: the tensor core adds the products of a block to the sum
    in one go, which loses at most a last place (2^-23) of the sum of magnitudes `size`; K / 16 blocks, and a few steps for scales and additions."""
    tol = (2.0 ** -8 if y.dtype == torch.bfloat16 else 0.0) * want.abs() + (K / 16 + 8) * 2.0 ** -23 * size + 1e-30
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} times what the roundings allow"


# ------------------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["normal", "wide", "ties", "extremes"])
@pytest.mark.parametrize("T,K", [(1, 32), (9, 96), (5, 2880), (130, 544), (3, 14336), (2, 20000 // 32 * 32)])
def test_rows(T, K, kind, dtype, form):
    x = rows_of(kind, T, K, dtype)
    want, got = fp4_matrix.quantize(x, form), ops.quantize_fp4(x.to(DEV), form)
    finite = torch.isfinite(x.float()).all(-1)
    # values, not bytes: a zero may carry either sign, and a block of zeros any scale
    nan_rows = lambda m: torch.nan_to_num(m.dequantize().cpu(), nan=7e30)
    assert torch.equal(nan_rows(got), nan_rows(want))
    assert torch.equal(torch.isnan(got.row_scales().cpu()), ~finite)
    assert torch.equal(got.dequantize(torch.bfloat16).cpu().nan_to_num(7.0), want.dequantize(torch.bfloat16).nan_to_num(7.0))


def test_rows_with_strides():
    x = rows_of("normal", 40, 704, torch.bfloat16).to(DEV)
    for v in (x[:, 64:320], x[::3, 1:257], x[:, :512].t()[:, :32]):
        assert torch.equal(ops.quantize_fp4(v).dequantize(), ops.quantize_fp4(v.contiguous().clone()).dequantize())
    assert ops.quantize_fp4(x[:0, :64]).dequantize().shape == (0, 64)


def test_padding_of_the_last_k_block_is_zero():
    m = ops.quantize_fp4(rows_of("normal", 3, 272, torch.bfloat16).to(DEV))
    c, s = fp4_matrix.Fp4Matrix(m.data, 3, 512, "nvfp4"), None
    assert not c.codes()[:, 272:].any() and not c.scales()[:, 17:].any()


# ------------------------------------------------------------------------------------------- products
SHAPES = [(1, 128, 64), (1, 6144, 4096), (2, 65, 96), (7, 4096, 14336), (16, 28672, 512), (17, 1000, 2880), (31, 200, 320), (33, 129, 256), (64, 4096, 1024), (65, 777, 288),
          (128, 512, 2048), (129, 640, 544), (200, 300, 1024), (256, 256, 256), (300, 5120, 2880), (513, 1111, 320), (777, 2880, 640), (1025, 4096, 512)]


@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_products(T, N, K, form):
    x = rows_of("wide" if T % 2 else "normal", T, K, torch.bfloat16).to(DEV)
    w = weight(N, K, form)
    xq, wq = ops.quantize_fp4(x, form).dequantize().double(), w.dequantize().double()
    want, size = xq @ wq.T, xq.abs() @ wq.abs().T
    close(ops.linear(x, w), want, size, K)
    close(ops.linear(x, w, out_fp32=True), want, size, K)
    g = torch.Generator().manual_seed(T)
    bias, res = torch.randn(N, generator=g).to(torch.bfloat16).to(DEV), torch.randn(T, N + 3, generator=g).to(DEV)[:, :N]
    want, size = want + bias.double() + res.double(), size + bias.double().abs() + res.double().abs()
    close(ops.linear(x, w, bias, res, out_fp32=True), want, size, K)
    rb = res.to(torch.bfloat16)
    close(ops.linear(x, w, bias, rb), want - res.double() + rb.double(), size, K)
    ops.check_kernel_status()


@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("T,N,K", [(1, 128, 64), (3, 1152, 2880), (16, 28672, 320), (40, 512, 1024), (150, 5760, 288), (300, 384, 512), (600, 1280, 2048)])
def test_gated_products(T, N, K, form):
    x = rows_of("normal", T, K, torch.bfloat16).to(DEV)
    w = weight(N, K, form, interleaved=True)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(DEV)
    xq, wq = ops.quantize_fp4(x, form).dequantize().double(), w.dequantize().double()
    y, size = xq @ wq.T + bias.double(), xq.abs() @ wq.abs().T + bias.double().abs()
    split = lambda t: (v.reshape(T, N // 2) for v in t.view(T, N // 128, 2, 64).unbind(2))
    (g, u), (sg, su) = split(y), split(size)
    got = ops.gate_up_act(x, w, bias).double()
    want = torch.nn.functional.silu(g) * u
    # silu's slope is at most 1.1; its own fp32 steps (an exponential and a division of a few last places each): 2^-20 of the result
    d = (K / 16 + 8) * 2.0 ** -23
    tol = 2.0 ** -8 * want.abs() + d * (1.1 * sg * (u.abs() + d * su) + g.abs() * su) + 2.0 ** -20 * want.abs() + 1e-30
    assert bool(((got - want).abs() <= tol).all())
    relu = ops.gate_up_act(x, w, bias, act="relu").double()
    rw = torch.relu(g) * u
    assert bool(((relu - rw).abs() <= 3 * 2.0 ** -8 * rw.abs() + 2 * d * (sg * (u.abs() + d * su) + g.abs() * su) + 1e-30).all())
    ops.check_kernel_status()


def test_quantised_rows_serve_several_products():
    x = rows_of("normal", 70, 576, torch.bfloat16).to(DEV)
    q = ops.quantize_fp4(x)
    for N in (64, 300):
        w = weight(N, 576, "nvfp4")
        assert torch.equal(ops.linear(q, w), ops.linear(x, w))


def test_rows_that_are_not_numbers_stay_to_themselves():
    for T in (5, 200):
        x = rows_of("normal", T, 512, torch.bfloat16).to(DEV)
        w = weight(256, 512, "nvfp4")
        ref = ops.linear(x, w)
        y = x.clone()
        y[1, 7], y[T - 2, 400] = math.inf, math.nan
        got = ops.linear(y, w)
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[1] = keep[T - 2] = False
        assert torch.equal(got[keep], ref[keep]) and bool(torch.isnan(got[~keep]).all())


def test_output_ranges_are_left_as_they_were():
    for T, N in ((3, 100), (140, 100)):
        x, w = rows_of("normal", T, 256, torch.bfloat16).to(DEV), weight(N, 256, "nvfp4")
        big = torch.full((T + 2, N + 7), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.linear(x, w, out=big[1:T + 1, 3:N + 3])
        assert torch.equal(big[1:T + 1, 3:N + 3], ops.linear(x, w))
        big[1:T + 1, 3:N + 3] = 3.0
        assert bool((big == 3.0).all())


def test_unaligned_rows_and_fp32_rows():
    for T in (4, 180):
        wide = rows_of("normal", T, 300, torch.bfloat16).to(DEV)
        w = weight(192, 256, "nvfp4")
        assert torch.equal(ops.linear(wide[:, 3:259], w), ops.linear(wide[:, 3:259].contiguous(), w))
        assert torch.equal(ops.linear(wide[:, :256].float(), w), ops.linear(wide[:, :256], w))


def test_same_results_every_time_and_from_graphs():
    for T, N, K in ((1, 512, 4096), (20, 640, 8192), (300, 1024, 1024)):
        x, w = rows_of("normal", T, K, torch.bfloat16).to(DEV), weight(N, K, "nvfp4")
        first = ops.linear(x, w)
        for _ in range(5):
            assert torch.equal(ops.linear(x, w), first)
        side = torch.cuda.Stream()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            side.wait_stream(torch.cuda.current_stream())
            with ops.graph_capture(g, stream=side):
                y = ops.linear(x, w)
            graphs.append((g, y))
        torch.cuda.synchronize()
        x2 = rows_of("normal", T, K, torch.bfloat16, seed=9).to(DEV)
        want = ops.linear(x2, w)
        x.copy_(x2)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, (g, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for _, y in graphs)


def test_refusals_of_device_tensors():
    w = weight(64, 64, "nvfp4")
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="different devices"):
        ops.linear(x.cpu(), w)
    with pytest.raises(ValueError, match="bias"):
        ops.linear(x, w, bias=torch.zeros(64, device=DEV))
    with pytest.raises(ValueError, match="output"):
        ops.linear(x, w, out=torch.zeros(2, 64, device=DEV))
    with pytest.raises(ValueError, match="residual"):
        ops.linear(x, w, residual=torch.zeros(2, 64, dtype=torch.float16, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_every_significand(dtype):
    """Blocks whose largest magnitude takes every significand of bf16 at many sizes under the row's largest, and whose other numbers are whole eighths of an
    e4m3 scale's significand times ties of e2m1, or next to those."""
    g = torch.Generator().manual_seed(12)
    rows, blocks = 128, 48
    x = torch.zeros(rows, blocks, 16)
    top = torch.arange(128, 256)[:, None] * 2.0 ** -torch.arange(blocks)[None, :].div(2, rounding_mode="floor").float()
    x[..., 0] = top * torch.where(torch.rand(rows, blocks, generator=g) < 0.5, -1.0, 1.0)
    tie = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])[torch.randint(0, 7, (rows, blocks, 15), generator=g)]
    scale = (top / 6).to(torch.float8_e4m3fn).float()[..., None]                       # (of a row scale of one; others move it by a power of two)
    near = (tie * scale).to(torch.bfloat16)
    bits = (near.view(torch.int16) + torch.randint(-1, 2, near.shape, generator=g).to(torch.int16)).clamp(min=0)
    x[..., 1:] = torch.minimum(bits.view(torch.bfloat16).float(), top[..., None]) * torch.where(torch.rand(rows, blocks, 15, generator=g) < 0.5, -1.0, 1.0)
    x = x.view(rows, -1).to(dtype)
    for row in (x, x * 2.0 ** 7, x * 2.0 ** -9):
        assert torch.equal(ops.quantize_fp4(row.to(DEV)).dequantize().cpu(), fp4_matrix.quantize(row, "nvfp4").dequantize())


@pytest.mark.parametrize("form", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,N,K", [(1, 128, 32), (1, 6144, 4096), (1, 28672, 4096), (1, 300, 8192), (1, 300, 16384), (1, 18944, 512), (2, 1000, 2880), (2, 6144, 4096),
                                   (2, 200, 8192), (3, 130, 288), (1, 14208, 6656)])
def test_rows_quantised_by_the_product(T, N, K, dtype, form):
    """Few rows that are not quantised yet: the same numbers as through the rows' own kernel, whichever of the two takes them."""
    wide = torch.full((T, K + 5), 9.0)
    wide[:, 1:K + 1] = rows_of("wide", T, K, torch.bfloat16).float()
    if T > 1:
        wide[1, 1 + K // 2] = math.nan
    x = wide.to(dtype).to(DEV)[:, 1:K + 1]
    w = weight(N, K, form)
    want = ops.linear(ops.quantize_fp4(x, form), w, out_fp32=True)
    for rows in (x, x.contiguous()):
        got = ops.linear(rows, w, out_fp32=True)
        assert torch.equal(got.nan_to_num(5.0), want.nan_to_num(5.0)) and torch.equal(torch.isnan(got), torch.isnan(want))
    gated = weight(128 * (N // 128), K, form, interleaved=True) if N >= 128 else None
    if gated is not None:
        assert torch.equal(ops.gate_up_act(x, gated).nan_to_num(5.0), ops.gate_up_act(ops.quantize_fp4(x, form), gated).nan_to_num(5.0))
    ops.check_kernel_status()


def test_rows_that_are_not_numbers_or_zero_and_the_product_that_quantises():
    w = weight(384, 512, "nvfp4")
    for fill in (0.0, math.inf, -math.inf, math.nan):
        x = rows_of("normal", 2, 512, torch.bfloat16).to(DEV)
        other = ops.linear(x, w)[0]
        x[1, 300:] = fill
        if fill == 0.0:
            x[1] = 0.0
        got = ops.linear(x, w)
        assert torch.equal(got[0], other) and bool((got[1] == 0).all() if fill == 0.0 else torch.isnan(got[1]).all())


def test_no_rows():
    w, gated = weight(192, 256, "nvfp4"), weight(256, 256, "nvfp4", interleaved=True)
    x = torch.zeros(0, 256, dtype=torch.bfloat16, device=DEV)
    for rows in (x, x.float(), ops.quantize_fp4(x)):
        assert ops.linear(rows, w).shape == (0, 192) and ops.gate_up_act(rows, gated).shape == (0, 128)


def test_offsets_beyond_32_bits():
    """2.2 G numbers: rows of them, weights of them, and the results of 2.2 G."""
    T, K = 66001, 32768
    big = torch.empty(T, K, dtype=torch.bfloat16, device=DEV)
    big.normal_(generator=torch.Generator(DEV).manual_seed(1))
    q = ops.quantize_fp4(big)
    last = ops.quantize_fp4(big[-70:])
    back = q.dequantize(torch.bfloat16)
    assert torch.equal(back[-70:], last.dequantize(torch.bfloat16)) and torch.equal(back[:3], ops.quantize_fp4(big[:3]).dequantize(torch.bfloat16))
    del back
    wq = last.dequantize().double()
    for rows in (1, 3, 70):                          # as weights
        x = rows_of("normal", rows, K, torch.bfloat16).to(DEV)
        xq = ops.quantize_fp4(x).dequantize().double()
        close(ops.linear(x, q)[:, -70:], xq @ wq.T, xq.abs() @ wq.abs().T, K)
    del big
    few = weight(128, K, "nvfp4")                    # as rows
    wq, xq = few.dequantize().double(), last.dequantize().double()
    close(ops.linear(q, few)[-70:], xq @ wq.T, xq.abs() @ wq.abs().T, K)
    del q
    x, w = rows_of("normal", 16800, 256, torch.bfloat16).to(DEV), weight(128256, 256, "mxfp4")
    y = ops.linear(x, w)[-5:]
    xq, wq = ops.quantize_fp4(x[-5:], "mxfp4").dequantize().double(), w.dequantize().double()
    close(y, xq @ wq.T, xq.abs() @ wq.abs().T, 256)
    ops.check_kernel_status()


@pytest.mark.parametrize("T,given", [(1, False), (2, False), (2, True), (20, True), (60, True)])
def test_parts_of_k_in_clusters_repeat(T, given):
    """Products whose parts of k meet in a cluster, a hundred in a row: the same sums every time."""
    x, w = rows_of("normal", T, 4096, torch.bfloat16).to(DEV), weight(640, 4096, "nvfp4")
    rows = ops.quantize_fp4(x) if given else x
    first = ops.linear(rows, w, out_fp32=True)
    xq, wq = ops.quantize_fp4(x).dequantize().double(), w.dequantize().double()
    close(first, xq @ wq.T, xq.abs() @ wq.abs().T, 4096)
    differs = torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(100):
        differs += (ops.linear(rows, w, out_fp32=True) != first).any()
    assert int(differs) == 0
    ops.check_kernel_status()


@pytest.mark.parametrize("T", [3, 40, 70, 200])
def test_results_near_the_smallest_normal_numbers(T):
    """Scales whose product is below the normal numbers, and results around their border: the same rules whichever kernel takes the rows."""
    N, K = 128, 256
    small = weight(N, K, "nvfp4")
    c = small.codes()
    w = ops.Fp4Matrix.from_codes(c[:, 0::2] | c[:, 1::2] << 4, small.scales(), small.row_scales() * 2.0 ** -58)
    x = (rows_of("normal", T, K, torch.float32) * 2.0 ** -66).to(DEV)
    xq, wq = ops.quantize_fp4(x).dequantize().double(), w.dequantize().double()
    want, size = xq @ wq.T, xq.abs() @ wq.abs().T
    assert float(want.abs().max()) > 2.0 ** -126
    # the bounds of `close`, and half a step of the subnormal numbers, 2^-150, for the result
    assert bool(((ops.linear(x, w, out_fp32=True).double() - want).abs() <= (K / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -150).all())


def test_a_norm_in_front_of_rows_of_either_type_and_stride():
    """norm_eps with fp32 rows, and with rows that do not lie together: the product of the normed rows."""
    T, K = 5, 512
    wide = rows_of("normal", T, K + 8, torch.float32).to(DEV) * 3.0
    w, gated = weight(192, K, "nvfp4"), weight(256, K, "nvfp4", interleaved=True)
    for dtype in (torch.float32, torch.bfloat16):
        x = wide.to(dtype)[:, 3:K + 3]
        xd = x.double()
        normed = xd * torch.rsqrt((xd * xd).mean(-1, keepdim=True) + 1e-5)
        rows = ops._normed_rows(x, 1e-5)
        # a sum of K squares, a root and a product in fp32, then the rows' type
        assert rows.dtype == dtype and bool(((rows.double() - normed).abs() <= ((K + 8) * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * normed.abs()).all())
        assert torch.equal(ops.linear(x, w, norm_eps=1e-5), ops.linear(rows, w)) and torch.equal(ops.gate_up_act(x, gated, norm_eps=1e-5), ops.gate_up_act(rows, gated))
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.linear(wide.half()[:, :K], w, norm_eps=1e-5)
