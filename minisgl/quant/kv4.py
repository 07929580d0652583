"""KV cache rows in 4 bits: codes under one 8-bit scale per 32 dims.

A group is 32 consecutive dims of one token's key (or value) in one KV head:

* scale s = (8 + m) 2^(e - 24), held as the byte 8 e + m (e 0..31, m 0..7): four
  significant bits between 2^-21 and 1920. s is the smallest such number with
  max |x| <= 7.5 s (the nearest end of the range beyond it);
* code c = clamp(round(x / s), -8, 7) + 8, rounded half to even; a NaN has
  code 8, the zero.

An element is s (c - 8): at most 4 + 4 significant bits, so every value is
exactly a bf16 number and no reader of the cache rounds it again. In the range
it is at most s / 2 from x, that is max |x| / 13.3 at worst (a scale is up to
1/8 above max |x| / 7.5).

A page of one head is one block of bytes, ``page_size * (d / 2 + d / 32)``
long: the codes, then the scales, in the order in which the attention kernel's
lanes take them as matrix fragments (d a multiple of 64, page_size of 16):

* K codes: rows of d / 2 bytes, one per token. A row is 32-bit words of eight
  dims 8 u .. 8 u + 7 (lowest nibble first); word u = 4 i + t stands at place
  t (d / 32) + i, so the d / 32 words of lane t are side by side, one per group.
* K scales: d / 32 bytes per token.
* V codes: rows of 2 d bytes, one per four tokens 4 a .. 4 a + 3. Dims 2 c
  (low nibble) and 2 c + 1 of the four tokens are one 32-bit word, whose bytes
  are tokens 0, 2, 1, 3; four words c = 4 x .. 4 x + 3 are a 16-byte chunk, and
  chunk x stands at place x ^ (2 (a mod 4)), which spreads the four rows that a
  warp reads at once over the shared-memory banks.
* V scales: d / 32 words per four tokens, bytes again for tokens 0, 2, 1, 3.
"""

from __future__ import annotations

import functools
from typing import Tuple

import torch

KV4_GROUP = 32
KV4_HEAD_DIMS = (64, 128)


def kv4_block_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one KV head (K or V)."""
    return page_size * (head_dim // 2 + head_dim // KV4_GROUP)


def kv4_check(page_size: int, head_dim: int) -> None:
    """Raise for a head dim or page size that the format does not have."""
    if head_dim not in KV4_HEAD_DIMS:
        raise ValueError(f"4-bit KV cache: head_dim must be one of {KV4_HEAD_DIMS}, got {head_dim}")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"4-bit KV cache: page_size must be a power of two >= 16, got {page_size}")


def kv4_scales(sf: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Scale bytes -> the scales they stand for."""
    sf = sf.to(torch.int32)
    return torch.ldexp((8 + sf % 8).to(dtype), sf // 8 - 24)


def quantize_kv4_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The format's statement: x [..., d] (any float type) -> (codes uint8
    [..., d], scale bytes uint8 [..., d / 32]), computed in float64."""
    b = x.double().unflatten(-1, (-1, KV4_GROUP))
    table = kv4_scales(torch.arange(256, device=x.device), torch.float64)
    amax = torch.where(b.isnan(), 0.0, b).abs().amax(-1)
    sf = torch.searchsorted(7.5 * table, amax.contiguous()).clamp(max=255)
    c = torch.round(b / table[sf][..., None]).nan_to_num(0.0, 7.0, -8.0).clamp(-8, 7) + 8
    return c.flatten(-2).to(torch.uint8), sf.to(torch.uint8)


def dequantize_kv4(codes: torch.Tensor, sf: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """(codes [..., d], scale bytes [..., d / 32]) -> values [..., d]."""
    v = (codes.float() - 8.0).unflatten(-1, (-1, KV4_GROUP)) * kv4_scales(sf)[..., None]
    return v.flatten(-2).to(dtype)


@functools.lru_cache(maxsize=32)
def _places(page_size: int, d: int, device: torch.device):
    """Byte places inside a block: K code bytes [page, d / 2], V code bytes
    [page, d / 2], K and V scale bytes [page, d / 32]."""
    groups, half = d // KV4_GROUP, d // 2
    tok = torch.arange(page_size, device=device)[:, None]
    c = torch.arange(half, device=device)[None]
    u = c // 4  # word of eight dims
    k = tok * half + ((u % 4) * groups + u // 4) * 4 + c % 4
    a, byte = tok // 4, torch.tensor([0, 2, 1, 3], device=device)[tok % 4]
    v = a * (2 * d) + ((c // 4) ^ (2 * (a % 4))) * 16 + (c % 4) * 4 + byte
    g = torch.arange(groups, device=device)[None]
    base = page_size * half
    return k, v, base + tok * groups + g, base + (a * groups + g) * 4 + byte


def pack_kv4(packed: torch.Tensor, sf: torch.Tensor) -> torch.Tensor:
    """Pages in plain order -> blocks: ``packed`` uint8 [2, ..., page, d / 2]
    (K, V; dim 2 i in the low nibble of byte i) and ``sf`` uint8
    [2, ..., page, d / 32] -> uint8 [2, ..., block bytes]."""
    page, d = packed.shape[-2], packed.shape[-1] * 2
    kv4_check(page, d)
    if packed.shape[0] != 2 or sf.shape != packed.shape[:-1] + (d // KV4_GROUP,):
        raise ValueError(f"pack_kv4: codes {tuple(packed.shape)} and scales {tuple(sf.shape)} do not belong together")
    out = torch.empty(packed.shape[:-2] + (kv4_block_bytes(page, d),), dtype=torch.uint8, device=packed.device)
    places = _places(page, d, packed.device)
    for kv in range(2):
        out[kv][..., places[kv].flatten()] = packed[kv].flatten(-2)
        out[kv][..., places[2 + kv].flatten()] = sf[kv].flatten(-2)
    return out


def unpack_kv4(blocks: torch.Tensor, page_size: int, head_dim: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Blocks [2, ..., block bytes] -> (packed [2, ..., page, d / 2], scale
    bytes [2, ..., page, d / 32]): the inverse of ``pack_kv4``."""
    kv4_check(page_size, head_dim)
    if blocks.shape[0] != 2 or blocks.shape[-1] != kv4_block_bytes(page_size, head_dim):
        raise ValueError(f"unpack_kv4: blocks {tuple(blocks.shape)} are not pages of {page_size} x {head_dim}")
    k, v, ks, vs = _places(page_size, head_dim, blocks.device)
    return (torch.stack([blocks[0][..., k], blocks[1][..., v]]),
            torch.stack([blocks[0][..., ks], blocks[1][..., vs]]))
