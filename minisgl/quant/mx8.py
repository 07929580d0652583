"""MXFP8 rows: E4M3 elements with one E8M0 scale per 32 columns, row-major.

A row-major tensor y [rows, cols] (cols a multiple of 32) becomes

* ``q`` uint8 [rows, cols]: E4M3 bits;
* ``sf`` uint8 [rows, cols / 32]: exponents (bias 127) of the blocks' scales.

Per block the scale is 2^e with the smallest e >= -126 for which max |y| <=
448 * 2^e, elements are y / 2^e rounded to nearest even. An all-zero block has
scale byte 0 and zero elements; a block with an infinity, a NaN or a magnitude
beyond float32 has scale byte 255 and NaN elements. The formats of the
block-scaled expert GEMM (``minisgl.quant.mxfp4``) hold the same numbers with
their scales blocked for the tensor cores; the reference has no 8-bit path.
"""

from __future__ import annotations

from typing import Tuple

import torch

MX8_BLOCK = 32
_E4M3_MAX = 448.0


def quantize_mx8_rows_reference(y: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The format's statement, in float64: y [rows, cols] -> (q, sf)."""
    rows, cols = y.shape
    if cols % MX8_BLOCK != 0:
        raise ValueError("MXFP8 rows: the width must be a multiple of 32")
    b = y.double().reshape(rows, cols // MX8_BLOCK, MX8_BLOCK)
    amax = b.abs().amax(-1)  # NaN where the block has one
    bad = ~(amax <= torch.finfo(torch.float32).max)
    amax = torch.where(bad, torch.ones_like(amax), amax)
    mant, ex = torch.frexp(amax)                      # amax = mant * 2^ex, mant in [0.5, 1)
    e = (ex - 9 + (mant > _E4M3_MAX / 512).int()).clamp(min=-126)
    zero = amax == 0
    t = b * torch.exp2(-e.double())[..., None]
    # E4M3 has steps of 2^-3 of a value's power of two, 2^-9 below 2^-6; torch rounds half to even
    power = torch.frexp(t)[1].clamp(min=-5) - 1
    step = torch.exp2((power - 3).double())
    t = torch.where(bad[..., None], torch.full_like(t, float("nan")), torch.round(t / step) * step)
    q = t.float().to(torch.float8_e4m3fn).view(torch.uint8)
    q = torch.where(bad[..., None], torch.full_like(q, 0x7F), torch.where(zero[..., None], torch.zeros_like(q), q))
    sf = torch.where(bad, 255, torch.where(zero, 0, e + 127)).to(torch.uint8)
    return q.reshape(rows, cols), sf


def dequantize_mx8_rows(q: torch.Tensor, sf: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """(q [rows, cols], sf [rows, cols / 32]) -> [rows, cols]."""
    rows, cols = q.shape
    vals = q.view(torch.float8_e4m3fn).double().reshape(rows, cols // MX8_BLOCK, MX8_BLOCK)
    scale = torch.exp2(sf.double() - 127.0)[..., None]
    scale = torch.where(sf[..., None] == 255, torch.full_like(scale, float("nan")), scale)
    return (vals * scale).reshape(rows, cols).to(dtype)
