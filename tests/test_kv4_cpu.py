"""The 4-bit KV cache on the CPU: format, layout, the operators' CPU path, refusals."""

import pytest
import torch

import kv4_oracle as oracle
from minisgl import ops
from minisgl.quant import dequantize_kv4, kv4_block_bytes, pack_kv4, quantize_kv4_reference, unpack_kv4


def test_scales_are_the_smallest_that_reach_and_values_are_bf16():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(400, 64, generator=g) * torch.exp2(torch.randint(-24, 16, (400, 1), generator=g))
    x[0] = 0
    x[1, 3] = 7.5 * 1.125  # exactly on a border
    codes, sf = quantize_kv4_reference(x)
    want_c, want_s = oracle.quantize(x)
    assert torch.equal(codes, want_c) and torch.equal(sf, want_s)
    table = oracle.scales(torch.arange(256))
    top = x.double().abs().view(400, 2, 32).amax(-1)
    s = table[sf.long()]
    inside = top <= 7.5 * 1920
    assert (7.5 * s >= top)[inside].all()
    below = table[(sf.long() - 1).clamp(min=0)]
    assert ((7.5 * below < top) | (sf == 0)).all()
    v = dequantize_kv4(codes, sf, torch.float64)
    assert torch.equal(v, v.to(torch.bfloat16).double())
    step = s.repeat_interleave(32, dim=-1).view(400, 64)
    keep = inside.repeat_interleave(32, dim=-1).view(400, 64)
    assert ((v - x.double()).abs() <= step / 2)[keep].all()
    assert torch.equal(v, oracle.values(codes[..., 0::2] | (codes[..., 1::2] << 4), sf))


def test_special_values_have_codes():
    x = torch.zeros(3, 32)
    x[0, 0], x[1, 0], x[2, 0], x[2, 1] = float("inf"), float("-inf"), float("nan"), 1.0
    v = dequantize_kv4(*quantize_kv4_reference(x))
    assert v[0, 0] == 7 * 1920 and v[1, 0] == -8 * 1920 and v[2, 0] == 0 and abs(v[2, 1] - 1) < 1 / 13


@pytest.mark.parametrize("page,d", [(16, 64), (64, 128), (256, 64)])
def test_blocks_hold_every_byte_once(page, d):
    packed = torch.randint(0, 256, (2, 3, 2, page, d // 2), dtype=torch.uint8)
    sf = torch.randint(0, 256, (2, 3, 2, page, d // 32), dtype=torch.uint8)
    blocks = pack_kv4(packed, sf)
    assert blocks.shape == (2, 3, 2, kv4_block_bytes(page, d))
    back = unpack_kv4(blocks, page, d)
    assert torch.equal(back[0], packed) and torch.equal(back[1], sf)
    assert blocks.int().sum() == packed.int().sum() + sf.int().sum()


def test_layout_of_single_elements():
    """Where the format says that a dim of a token lies."""
    page, d = 32, 128
    for tok, dim in [(0, 0), (5, 1), (6, 40), (7, 127), (30, 77)]:
        packed = torch.zeros(2, page, d // 2, dtype=torch.uint8)
        packed[:, tok, dim // 2] = 15 << (4 * (dim % 2))
        sf = torch.zeros(2, page, 4, dtype=torch.uint8)
        sf[:, tok, dim // 32] = 9
        k, v = pack_kv4(packed, sf)
        u = dim // 8
        at = tok * 64 + 4 * ((u % 4) * 4 + u // 4) + dim % 8 // 2
        assert k[at] == 15 << (4 * (dim % 2)) and k[2048 + tok * 4 + dim // 32] == 9 and (k != 0).sum() == 2
        row, byte, c = tok // 4, [0, 2, 1, 3][tok % 4], dim // 2
        at = row * 256 + 16 * ((c // 4) ^ (2 * (row % 4))) + 4 * (c % 4) + byte
        assert v[at] == 15 << (4 * (dim % 2)) and v[2048 + 4 * (row * 4 + dim // 32) + byte] == 9 and (v != 0).sum() == 2


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
def test_operators_on_the_cpu(d, page):
    hq, hk = 6, 2
    lens, queries = [40, 3, 0, 17], [4, 5, 1, 1]
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page)
    q = torch.randn(sum(queries), hq * d)
    seq = torch.tensor(lens, dtype=torch.int32)
    cu = torch.tensor([0] + list(torch.tensor(queries).cumsum(0)), dtype=torch.int32)
    got = ops.prefill_attention_kv4(q, pool, 1, table, rows, seq, cu, 5, hq, hk, d, page, 0.1)
    want, _ = oracle.attention(q.double().view(-1, hq, d), packed, sf, 1, table, rows, lens, queries, hq, hk, 0.1)
    torch.testing.assert_close(got.double().view_as(want), want, atol=1e-5, rtol=1e-5)
    out = torch.empty(4, hq * d)
    ops.decode_attention_kv4(q[:4], pool, 1, table, rows, seq, hq, hk, d, page, 0.1, out=out)
    want, _ = oracle.attention(q[:4].double().view(-1, hq, d), packed, sf, 1, table, rows, lens, [1] * 4, hq, hk, 0.1)
    torch.testing.assert_close(out.double().view_as(want), want, atol=1e-5, rtol=1e-5)

    cs = oracle.cos_sin(64, d)
    qkv = torch.randn(3, (hq + 2 * hk) * d)
    w = 1 + 0.1 * torch.randn(d)
    slots = torch.tensor([page, 2, 2 * page + 5], dtype=torch.int32)
    keep = qkv.clone()
    ops.rope_store_kv4(qkv, torch.tensor([0, 63, 9]), cs, w, None, pool, 0, slots, hq, hk, d, page, 1e-6)
    x = keep.view(3, hq + 2 * hk, d)
    pos = torch.tensor([0, 63, 9])
    torch.testing.assert_close(qkv[:, :hq * d].double().view(3, hq, d), oracle.rope_rows(x[:, :hq], w, cs[pos]),
                               atol=1e-5, rtol=1e-5)
    assert torch.equal(qkv[:, hq * d:], keep[:, hq * d:])
    k, v = ops.load_kv4(pool, 0, slots, hk, d, page, torch.float64)
    c, byte = oracle.quantize(x[:, hq + hk:])
    assert torch.equal(v, oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte))
    kr = oracle.rope_rows(x[:, hq:hq + hk], None, cs[pos])
    top = kr.abs().reshape(3, hk, -1, 32).amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(kr.shape)
    assert ((k - kr).abs() <= top * (1.125 / 15 + 1e-5)).all()


def test_copy_pages_on_the_cpu():
    pool = torch.randint(0, 256, (2, 3, 9, 2, 16 * 34), dtype=torch.uint8)
    want = pool.clone()
    want[:, :, [4, 5, 0]] = pool[:, :, [1, 1, 8]]
    assert torch.equal(ops.copy_pages(pool, [1, 1, 8], torch.tensor([4, 5, 0])), want)
    latent = torch.randn(2, 5, 16, 24)
    want = latent.clone()
    want[:, 4] = latent[:, 3]
    assert torch.equal(ops.copy_pages(latent, [3, 2], [4, 2], page_dim=1), want)


@pytest.mark.parametrize("src,dst,error", [
    ([0], [9], IndexError), ([-1], [2], IndexError), ([0, 1], [2], ValueError), ([0, 1], [2, 2], ValueError),
    ([0, 2], [2, 3], ValueError), ([3, 3], [3, 3], ValueError), (torch.tensor([1.0]), [2], ValueError), ([0.5], [2], TypeError)])
def test_copy_pages_refuses(src, dst, error):
    pool = torch.zeros(2, 3, 9, 2, 16, dtype=torch.uint8)
    with pytest.raises(error):
        ops.copy_pages(pool, src, dst)


def test_refusals_on_the_cpu():
    d, hk, page = 64, 2, 16
    pool = torch.zeros(2, 1, 4, hk, kv4_block_bytes(page, d), dtype=torch.uint8)
    x, i3 = torch.zeros(3, hk * d), torch.zeros(3, dtype=torch.int32)
    pt, q = torch.zeros(3, 64, dtype=torch.int32), torch.zeros(3, 4 * d)
    bad = [
        lambda: ops.store_kv4(x, x[:2], pool, 0, i3, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 1, i3, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3 + 64, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3 - 1, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3, hk, d, 24),
        lambda: ops.store_kv4(x, x, pool, 0, i3, hk, 96, page),
        lambda: ops.store_kv4(x, x, pool.float(), 0, i3, hk, d, page),
        lambda: ops.load_kv4(pool, 0, i3 + 64, hk, d, page),
        lambda: ops.load_kv4(pool, -1, i3, hk, d, page),
        lambda: ops.rope_store_kv4(q, i3, oracle.cos_sin(8, d), None, None, pool, 0, i3, 4, hk, d, page, 1e-6),
        lambda: ops.rope_store_kv4(torch.zeros(3, 8 * d), i3, oracle.cos_sin(8, 32), None, None, pool, 0, i3, 4, hk, d,
                                   page, 1e-6),
        lambda: ops.rope_store_kv4(torch.zeros(3, 8 * d), i3, oracle.cos_sin(8, d), None, None, pool, 0, i3, 4, hk, d,
                                   page, 1e-6, q_out=q[:1].expand(3, -1)),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3, 3, hk, d, page, 0.1),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3, 4, hk, d, page, -0.1),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3, 8, hk, d, page, 0.1),
        lambda: pack_kv4(torch.zeros(2, 16, 32, dtype=torch.uint8), torch.zeros(2, 16, 1, dtype=torch.uint8)),
        lambda: unpack_kv4(pool, 32, d),
    ]
    for call in bad:
        with pytest.raises((ValueError, IndexError)):
            call()
