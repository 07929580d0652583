"""4-bit weights with group scales for the dense projections.

A weight W [N, K] is stored as codes c in 0..15 with one scale (and
optionally one zero point) per row and group of ``group`` columns:

    W[n, k] = (c[n, k] - z[n, k // group]) * s[n, k // group]

z is 8 where a weight has no zero points (symmetric quantisation). Groups are
32, 64 or 128 columns; the last one may be short (K a multiple of 8). This is
the form in which group-quantised checkpoints come: ``int4_weight`` takes the
codes packed two per byte and lays them out once for the kernels
(``minisgl/csrc/int4.cu``); ``quantize_int4`` makes them from a float weight.

Layout. Rows are cut into tiles of 16, columns into blocks of 64, both an even
number (rows are padded to 32, columns to 128); tile and block fill 512 bytes,
16 for each lane of a warp. Lane 4 g + t holds columns 4 t .. 4 t + 3 of each 16
of rows g and g + 8, in four words; word j has columns 16 j + 4 t + 2 p + e of
row g + 8 h at bit 4 (4 e + 2 p + h), as c - 8 in two's complement. A byte's
upper half is thus a signed code of row g + 8 (of row g after a shift by 4), and
a word gives two of the four registers (four 8-bit values each) that a warp-level
16 x 8 x 32 product takes of its first operand; unpacked to pairs of 16-bit
values, it is what a lane stores into 16 rows x 8 columns of tensor memory. A
word's columns lie under one group. Scales are [tile, group, g, h], so that a lane's two are one
word, zero points [tile, group, g] with z[g] | z[g + 8] << 4. Padding rows and
columns have scale 0.

The reference has no weight quantisation; its projections run bf16 library
GEMMs (python/minisgl/layers/linear.py:13-127).
"""

from __future__ import annotations

from typing import Optional

import torch

GROUPS = (32, 64, 128)
MAX_SCALE = 2.0 ** 90  # times a group's integer sum, 2^37 at most, it is still a float32 (products of few rows)
_TILE, _BLOCK, _STEP = 16, 64, 128  # rows are padded to two tiles, columns to a step


@torch.inference_mode(False)
@torch.no_grad()
def _ordinary(t: torch.Tensor) -> torch.Tensor:
    return t.clone() if t.is_inference() else t


def _tiles(n: int) -> int:
    return 2 * -(-n // (2 * _TILE))


class Int4Weight:
    """A 4-bit weight in the kernels' layout (made by ``int4_weight`` or
    ``quantize_int4``): ``packed`` uint8 [tiles, 2 ceil(K / 128), 512],
    ``scales`` bf16 / fp16 [tiles, groups, 8, 2] and ``zeros`` uint8
    [tiles, groups rounded up to even, 8] or None, tiles = 2 ceil(N / 32), groups =
    128 ceil(K / 128) / group;
    ``row_pow`` float32 [16 tiles]: a power of two near 2^-11 of a row's largest scale
    (1 where that is 0), which fp16 products take out of the row. The parts are not
    replaced, since the native handle and captured graphs hold them; ``copy_`` puts
    another weight of the same form into them. What is written to ``scales`` by hand
    (by torch: a tensor's version shows it) the calls after it see; a graph captured
    before sees it too, but keeps fp16 rows' powers, so there ``copy_`` is the way."""

    __slots__ = ("_packed", "_scales", "_zeros", "_row_pow", "_n", "_k", "_group", "_handle", "_version")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor],
                 row_pow: torch.Tensor, n: int, k: int, group: int) -> None:
        # tensors of inference mode have no version, and are not written outside of it
        packed, scales, zeros, row_pow = (t if t is None else _ordinary(t) for t in (packed, scales, zeros, row_pow))
        self._packed, self._scales, self._zeros, self._row_pow = packed, scales, zeros, row_pow
        self._n, self._k, self._group = n, k, group
        self._handle = None
        self._version = scales._version  # of the scales that row_pow is of
        if packed.is_cuda:
            self.native()  # checked, and its device's error word made, here and not inside somebody's graph capture

    packed = property(lambda self: self._packed)
    scales = property(lambda self: self._scales)
    zeros = property(lambda self: self._zeros)
    n = property(lambda self: self._n)
    k = property(lambda self: self._k)
    group = property(lambda self: self._group)

    @property
    def row_pow(self) -> torch.Tensor:
        return self._row_pow if self._scales._version == self._version else _row_powers(self._scales)

    def native(self, powers: bool = False):
        """The weight as one argument of the native calls (made with a CUDA weight). ``powers``: for calls that read the
        rows' powers; where the scales were written since, with powers of this call's own."""
        if powers and self._scales._version != self._version:
            return self._native_with(self.row_pow)
        if self._handle is None:
            self._handle = self._native_with(self._row_pow)
        return self._handle

    def _native_with(self, row_pow: torch.Tensor):
        from minisgl import ops

        return ops.native().Int4Handle(self.packed, self.scales, self.zeros, row_pow, self.n, self.k, self.group,
                                       ops.error_word(self.device))

    def copy_(self, src: "Int4Weight") -> "Int4Weight":
        """Put the values of ``src`` (same n, k, group, type of the scales, and zero points or none) into this
        weight's parts, which captured graphs go on reading."""
        if not isinstance(src, Int4Weight) or self._form() != src._form():
            raise ValueError("Int4Weight.copy_: another weight of the same n, k, group and scale type, "
                             "with zero points where this one has them")
        self._packed.copy_(src.packed)
        self._scales.copy_(src.scales)
        if self._zeros is not None:
            self._zeros.copy_(src.zeros)
        self._row_pow.copy_(src.row_pow)
        self._version = self._scales._version
        return self

    def _form(self):
        return self.n, self.k, self.group, self.scales.dtype, self.zeros is not None

    def __reduce__(self):
        return Int4Weight, (self.packed, self.scales, self.zeros, self.row_pow, self.n, self.k, self.group)

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def to(self, device) -> "Int4Weight":
        device = torch.device(device)  # not a type: the parts keep theirs
        zeros = None if self.zeros is None else self.zeros.to(device)
        return Int4Weight(self.packed.to(device), self.scales.to(device), zeros, self.row_pow.to(device), self.n,
                          self.k, self.group)


def _tile_rows(t: torch.Tensor, groups: int) -> torch.Tensor:
    """[N, groups of K] -> [tiles, groups, 8, 2] (row g + 8 h at [g, h]), padded with zeros."""
    n, g = t.shape
    tiles = _tiles(n)
    full = t.new_zeros(tiles * _TILE, groups)
    full[:n, :g] = t
    return full.view(tiles, 2, 8, groups).permute(0, 3, 2, 1).contiguous()


def _row_powers(tiled: torch.Tensor) -> torch.Tensor:
    """Scales [tiles, groups, 8, 2] -> 2^-11 of the power of two at or below each row's largest (not below 2^-126, whose
    inverse is a float32), 1 where that is 0 or not finite. Under it the row's scales are below 2^12, 15 of which fp16
    holds, and those down to 2^-25 of the largest keep all of their bits."""
    top = tiled.float().abs().amax(1).transpose(1, 2).reshape(-1)  # [tile, g, h] -> row
    live = (top > 0) & (top <= torch.finfo(torch.float32).max)
    power = (top.view(torch.int32) & 0x7F800000).view(torch.float32)  # the exponent's bits alone
    return torch.where(live, (power * 2.0 ** -11).clamp(min=2.0 ** -126), 1.0)


def _pack_reference(codes: torch.Tensor) -> torch.Tensor:
    """The layout's statement: codes [N, K / 2] -> packed [tiles, blocks, 512]."""
    n, k = codes.shape[0], 2 * codes.shape[1]
    tiles, blocks = _tiles(n), 2 * -(-k // _STEP)
    if tiles * _TILE != n or blocks * _BLOCK != k:
        full = codes.new_zeros(tiles * _TILE, blocks * _BLOCK // 2)
        full[:n, : k // 2] = codes
    else:
        full = codes
    # byte b of a row holds columns 2b (e = 0) and 2b + 1 (e = 1): [tile, h, g, block, j, t, p]
    c = full.view(tiles, 2, 8, blocks, 4, 4, 2).permute(1, 0, 3, 2, 5, 4, 6)  # [h, tile, block, g, t, j, p]
    top, low = c[0], c[1]
    # bytes of a word: (e, p) from the lowest; the nibbles of a byte: h
    packed = torch.empty(tiles, blocks, 8, 4, 4, 2, 2, dtype=torch.uint8, device=codes.device)
    packed[..., 0, :] = (top & 15) | (low << 4)
    packed[..., 1, :] = (top >> 4) | (low & 0xF0)
    packed ^= 0x88  # c - 8, two's complement
    return packed.view(tiles, blocks, 512)


@torch.inference_mode(False)
@torch.no_grad()
def int4_weight(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                group: int = 128) -> Int4Weight:
    """``codes`` uint8 [N, K / 2] (column 2i in the low nibble of byte i),
    ``scales`` bf16 / fp16 [N, ceil(K / group)], finite and not above 2^90,
    ``zeros`` uint8 (0..15) of the same shape or None (8 everywhere) -> the
    kernels' layout, on the same device."""
    if codes.dim() != 2 or codes.dtype != torch.uint8:
        raise ValueError("int4_weight: codes must be uint8 [N, K / 2]")
    n, k = codes.shape[0], 2 * codes.shape[1]
    if group not in GROUPS:
        raise ValueError(f"int4_weight: group of 32, 64 or 128, got {group}")
    if n == 0 or k == 0 or k % 8 != 0:
        raise ValueError(f"int4_weight: N >= 1 and K a positive multiple of 8, got N={n}, K={k}")
    shape = (n, -(-k // group))
    if tuple(scales.shape) != shape or scales.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"int4_weight: scales must be bf16 or fp16 {shape}, got {scales.dtype} {tuple(scales.shape)}")
    if zeros is not None and (tuple(zeros.shape) != shape or zeros.dtype != torch.uint8):
        raise ValueError(f"int4_weight: zeros must be uint8 {shape}, got {zeros.dtype} {tuple(zeros.shape)}")
    if any(t.device != codes.device for t in (scales, zeros) if t is not None):
        raise ValueError("int4_weight: codes, scales and zeros must be on one device")
    if zeros is not None and bool((zeros > 15).any()):
        raise ValueError("int4_weight: zero points must be 0..15")
    if not bool((scales.abs() <= (MAX_SCALE if scales.dtype == torch.bfloat16 else 65504.0)).all()):
        raise ValueError("int4_weight: scales must be finite and not above 2^90 in magnitude")
    if codes.is_cuda:
        from minisgl import ops

        ops._count()
        packed = ops.native().int4_pack(codes if codes.stride(1) == 1 else codes.contiguous())
    else:
        packed = _pack_reference(codes)
    blocks = packed.shape[1]
    groups = blocks * _BLOCK // group
    z = None
    if zeros is not None:
        z = _tile_rows(zeros, groups + groups % 2)  # whole 16-byte rows
        z = z[..., 0] | (z[..., 1] << 4)
    tiled = _tile_rows(scales, groups)
    return Int4Weight(packed, tiled, z, _row_powers(tiled), n, k, group)


def int4_codes(w: Int4Weight) -> torch.Tensor:
    """The codes of a weight, uint8 [N, K]."""
    tiles, blocks = w.packed.shape[:2]
    b = (w.packed ^ 0x88).view(tiles, blocks, 8, 4, 4, 2, 2)  # [tile, block, g, t, j, e, p]
    c = torch.stack([b & 15, b >> 4], dim=-1)        # ..., h
    c = c.permute(0, 7, 2, 1, 4, 3, 6, 5)            # [tile, h, g, block, j, t, p, e]
    return c.reshape(tiles * _TILE, blocks * _BLOCK)[: w.n, : w.k]


def dequantize_int4(w: Int4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The weight as [N, K], (c - z) * s computed in float64 and rounded once."""
    c = int4_codes(w).double()
    of = torch.arange(w.k, device=w.device) // w.group

    def spread(t: torch.Tensor) -> torch.Tensor:  # [tile, group, g, h] -> [N, K]
        return t.permute(0, 3, 2, 1).reshape(-1, t.shape[1])[: w.n].double()[:, of]

    z = 8.0 if w.zeros is None else spread(torch.stack([w.zeros & 15, w.zeros >> 4], dim=-1))
    return ((c - z) * spread(w.scales)).to(dtype)


def quantize_int4(w: torch.Tensor, group: int = 128, symmetric: bool = True,
                  scale_dtype: torch.dtype = torch.bfloat16) -> Int4Weight:
    """Round-to-nearest quantisation of a float weight [N, K]. Symmetric: scale
    max |w| / 7, codes 1..15 around 8. Otherwise the group's range (widened to
    hold 0) over 15 steps, with the zero point at the code that stands for 0."""
    n, k = w.shape
    if group not in GROUPS:
        raise ValueError(f"quantize_int4: group of 32, 64 or 128, got {group}")
    if n == 0 or k == 0 or k % 8 != 0:
        raise ValueError(f"quantize_int4: N >= 1 and K a positive multiple of 8, got N={n}, K={k}")
    groups = -(-k // group)
    x = w.new_zeros(n, groups * group, dtype=torch.float32)
    x[:, :k] = w
    x = x.view(n, groups, group)
    if symmetric:
        scales = (x.abs().amax(-1) / 7.0).to(scale_dtype)
        zeros = None
        z = torch.full_like(scales, 8.0, dtype=torch.float32)
    else:
        lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        scales = ((hi - lo) / 15.0).to(scale_dtype)
        live = torch.where(scales > 0, scales.float(), torch.ones_like(lo))
        z = (-lo / live).round().clamp(0, 15)
        zeros = z.to(torch.uint8)
    live = torch.where(scales > 0, scales.float(), torch.ones_like(z))
    c = (x / live[..., None]).round().add(z[..., None]).clamp(0, 15).to(torch.uint8).view(n, -1)[:, :k]
    return int4_weight(c[:, 0::2] | (c[:, 1::2] << 4), scales, zeros, group)
