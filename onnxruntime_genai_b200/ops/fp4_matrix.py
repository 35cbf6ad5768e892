"""Matrices of 4-bit floating-point numbers: e2m1 codes in blocks along K that share a scale (NVFP4: blocks of 16, e4m3; MXFP4: blocks of 32, a power
of two), one fp32 scale per row, in the layout of csrc/fp4_matrix.cuh.

`Fp4Matrix.from_codes(codes, scales, scale)` lays out a checkpoint's weight once at load time; `ops.quantize_fp4(x)` makes one of a step's rows.
`ops.linear` and `ops.gate_up_act` accept an Fp4Matrix as the weight (the rows are then quantised in its form, and both operands stay 4 bits wide) and, with
it, as the rows.  `dequantize()` gives the numbers that it stands for.

Reference semantics of the weights: MatMulBlockQuantizedFp4Weight as emitted by src/python/py/models/builders/base.py:1919-1949 (codes [N, K/2] with
the even k in the low half of a byte, e4m3 scales [N, K/16], one fp32 scale).
"""
from __future__ import annotations

from typing import Optional

import torch

FORMS = {"nvfp4": 0, "mxfp4": 1}
BLOCK = {"nvfp4": 16, "mxfp4": 32}
LARGEST = {"nvfp4": 0x7e, "mxfp4": 0xfe}   # bytes of block scales: 0x7f and 0xff are not numbers, and e4m3 scales have no sign
KB = 256                                   # k values of a k-block
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _padded(rows: int) -> int:
    return (rows + 127) // 128 * 128


def sizes(rows: int, K: int, form: str):
    """Bytes of the codes, of the block scales and of the row scales."""
    kb, p = (K + KB - 1) // KB, _padded(rows)
    return kb * p * 128, kb * p * (KB // BLOCK[form]), 4 * p


def matrix_bytes(rows: int, K: int, form: str) -> int:
    return _padded(rows) * ((K + KB - 1) // KB * (128 + KB // BLOCK[form]) + 4)


def swizzle(device) -> torch.Tensor:
    """[8, 8]: the chunk that stands at a place of a row, by row % 8 (its own inverse)."""
    i = torch.arange(8, device=device)
    return i[:, None] ^ i[None, :]


def e2m1_codes(v: torch.Tensor) -> torch.Tensor:
    """Codes of values that are already over their scale: nearest, ties to the even code, at most 6."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return c + 8 * ((v < 0) & (c > 0)).to(torch.uint8)


def e2m1_values(c: torch.Tensor) -> torch.Tensor:
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=c.device)
    return table[c.int()]


def block_scales(scales: torch.Tensor, form: str) -> torch.Tensor:
    """fp32 values of the bytes of block scales."""
    if form == "nvfp4":
        return scales.view(torch.float8_e4m3fn).float()
    return torch.ldexp(torch.ones(scales.shape, dtype=torch.float32, device=scales.device), scales.int() - 127)


class Fp4Matrix:
    """[rows, K] numbers; `data` is the one buffer that the kernels read."""
    __slots__ = ("data", "rows", "K", "form", "interleaved")
    dtype = torch.bfloat16

    def __init__(self, data: torch.Tensor, rows: int, K: int, form: str, interleaved: bool = False):
        self.data, self.rows, self.K, self.form = data, rows, K, form
        self.interleaved = interleaved          # weights of gate_up_act: blocks of 64 gate rows + 64 up rows

    @property
    def shape(self):
        return (self.rows, self.K)

    @property
    def device(self):
        return self.data.device

    @property
    def is_cuda(self):
        return self.data.is_cuda

    @staticmethod
    def check(rows: int, K: int, form: str) -> None:
        if form not in FORMS:
            raise ValueError(f"4-bit form {form!r}: one of {', '.join(FORMS)} is wanted")
        if rows < 0 or K <= 0 or K % BLOCK[form]:
            raise ValueError(f"{form}: {rows} rows of {K}: whole blocks of {BLOCK[form]} are wanted")

    @staticmethod
    def from_codes(codes: torch.Tensor, scales: torch.Tensor, scale: Optional[torch.Tensor] = None, form: str = "nvfp4", device=None,
                   interleaved: bool = False) -> "Fp4Matrix":
        """codes uint8 [N, K/2] (the even k in the low half of a byte); scales [N, K/block]: bytes, or float8_e4m3fn; scale: fp32, one number, one per row
        ([N]), or None (1).  Scales that are not numbers, or negative, are refused.  The layout is made where `codes` lives and moved to `device`.  interleaved: the rows are in interleave_gate_up's order."""
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise ValueError("codes are uint8 [N, K/2]")
        N, K = codes.shape[0], codes.shape[1] * 2
        Fp4Matrix.check(N, K, form)
        per = K // BLOCK[form]
        scales = scales.view(torch.uint8) if scales.dtype != torch.uint8 else scales
        if scales.shape != (N, per):
            raise ValueError(f"block scales have the shape {tuple(scales.shape)}: {(N, per)} is wanted")
        if bool((scales > LARGEST[form]).any()):
            raise ValueError(f"a block scale of {int(scales.max()):#x}: {form} scales are numbers without a sign, bytes up to {LARGEST[form]:#x}")
        if scale is not None and scale.numel() not in (1, N):
            raise ValueError(f"{scale.numel()} scales for {N} rows")
        if interleaved and N % 128:
            raise ValueError("interleaved gate and up rows come in blocks of 64 + 64")
        dev, kb, p, nb = codes.device, (K + KB - 1) // KB, _padded(N), KB // BLOCK[form]
        n_codes, n_scales, _ = sizes(N, K, form)
        data = torch.zeros(matrix_bytes(N, K, form), dtype=torch.uint8, device=dev)
        c = torch.zeros(p, kb * 128, dtype=torch.uint8, device=dev)
        c[:N, :K // 2] = codes
        c = c.view(p // 8, 8, kb, 8, 16)
        r = torch.arange(8, device=dev)[:, None]
        c = c.permute(1, 3, 2, 0, 4)[r, swizzle(dev)]                      # [row % 8, place, k-block, row / 8, 16]
        data[:n_codes].view(kb, p // 8, 8, 8, 16).copy_(c.permute(2, 3, 0, 1, 4))
        s = torch.zeros(p, kb * nb, dtype=torch.uint8, device=dev)
        s[:N, :per] = scales.to(dev)
        s = s.view(p // 128, 4, 32, kb, nb // 4, 4).permute(3, 0, 4, 2, 1, 5)
        data[n_codes:n_codes + n_scales].view(kb, p // 128, nb // 4, 32, 4, 4).copy_(s)
        rs = data[n_codes + n_scales:].view(torch.float32)
        rs[:N] = 1.0 if scale is None else scale.float().to(dev).reshape(-1)
        return Fp4Matrix(data if device is None else data.to(device), N, K, form, interleaved)

    def codes(self) -> torch.Tensor:
        """uint8 [rows, K], one code each."""
        kb, p = (self.K + KB - 1) // KB, _padded(self.rows)
        c = self.data[:sizes(*self.shape, self.form)[0]].view(kb, p // 8, 8, 8, 16).permute(2, 3, 0, 1, 4)
        r = torch.arange(8, device=self.device)[:, None]
        c = c[r, swizzle(self.device)].permute(3, 0, 2, 1, 4).reshape(p, kb * 128)[:self.rows, :self.K // 2]
        return torch.stack([c & 0xF, c >> 4], dim=-1).flatten(1)

    def scales(self) -> torch.Tensor:
        """uint8 [rows, K/block]."""
        n_codes, n_scales, _ = sizes(*self.shape, self.form)
        kb, p, nb = (self.K + KB - 1) // KB, _padded(self.rows), KB // BLOCK[self.form]
        s = self.data[n_codes:n_codes + n_scales].view(kb, p // 128, nb // 4, 32, 4, 4).permute(1, 4, 3, 0, 2, 5)
        return s.reshape(p, kb * nb)[:self.rows, :self.K // BLOCK[self.form]].contiguous()

    def row_scales(self) -> torch.Tensor:
        """fp32 [rows]."""
        n_codes, n_scales, _ = sizes(*self.shape, self.form)
        return self.data[n_codes + n_scales:].view(torch.float32)[:self.rows]

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """[rows, K] as `dtype` (fp32 or bf16): the kernel on CUDA devices, else its restatement."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"4-bit numbers are read back as float32 or bfloat16, not {dtype}")
        if self.is_cuda:
            from . import _dequantize_fp4
            return _dequantize_fp4(self, dtype)
        sc = block_scales(self.scales(), self.form)
        v = e2m1_values(self.codes()).view(*sc.shape, BLOCK[self.form]) * sc[..., None] * self.row_scales()[:, None, None]
        return v.view(self.rows, self.K).to(dtype)


def quantize(x: torch.Tensor, form: str) -> Fp4Matrix:
    """What csrc/quantize_fp4.cu computes, in torch (the CPU path)."""
    rows, K = x.shape
    b = x.float().view(rows, K // BLOCK[form], BLOCK[form])
    bad = ~torch.isfinite(x.float()).all(-1)
    b = torch.where(bad[:, None, None], torch.zeros_like(b), b)
    top = b.abs().amax(-1)
    if form == "nvfp4":
        m, e = torch.frexp(top.amax(-1, keepdim=True))
        e = torch.where(m <= 1.3125 / 2, e - 12, e - 11).clamp(min=-100)
        b = torch.ldexp(b, -e[..., None])
        s8 = (torch.ldexp(top, -e) / torch.full_like(top, 6.0)).to(torch.float8_e4m3fn)
        sc = s8.float()[..., None]
        c, scales, row = e2m1_codes(torch.where(sc > 0, b / sc, torch.zeros_like(b))), s8.view(torch.uint8), torch.ldexp(torch.ones(rows), e[:, 0])
    else:
        e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(min=-127)
        c, scales, row = e2m1_codes(torch.ldexp(b, -e[..., None])), (e + 127).to(torch.uint8), torch.ones(rows)
    c = c.view(rows, K)
    return Fp4Matrix.from_codes(c[:, 0::2] | (c[:, 1::2] << 4), scales, torch.where(bad, torch.full_like(row, float("nan")), row), form)
