"""4-bit group-scaled weights and MXFP8 rows on the CPU: layouts, formats, the
restatements that the GPU tests compare with, and the refusals."""

import math

import pytest
import torch

from minisgl import ops
from minisgl.quant import (dequantize_int4, dequantize_mx8_rows, int4_codes, int4_weight, quantize_int4,
                           quantize_mx8_rows_reference)


def _weight(n, k, group, zeros, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, -(-k // group), generator=g) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z, int4_weight(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, z, group)


@pytest.mark.parametrize("n,k,group", [(16, 64, 64), (1, 8, 32), (17, 72, 32), (40, 200, 128), (33, 192, 64)])
@pytest.mark.parametrize("zeros", [False, True])
def test_int4_layout_keeps_codes(n, k, group, zeros):
    codes, scales, z, w = _weight(n, k, group, zeros)
    assert torch.equal(int4_codes(w), codes)
    want = torch.empty(n, k, dtype=torch.float64)
    for j in range(k):
        zj = z[:, j // group].double() if zeros else 8.0
        want[:, j] = (codes[:, j].double() - zj) * scales[:, j // group].double()
    assert torch.equal(dequantize_int4(w, torch.float64), want)


def test_int4_layout_words():
    """One code at a time: where the layout's description puts it."""
    n, k = 32, 128
    for row, col in [(0, 0), (5, 3), (8, 1), (15, 63), (16, 64), (27, 101)]:
        codes = torch.zeros(n, k, dtype=torch.uint8)
        codes[row, col] = 13
        w = int4_weight(codes[:, 0::2] | (codes[:, 1::2] << 4), torch.ones(n, 2, dtype=torch.bfloat16), None, 64)
        tile, r, block, c = row // 16, row % 16, col // 64, col % 64
        h, g, j, t, p, e = r // 8, r % 8, c // 16, c % 16 // 4, c % 4 // 2, c % 2
        words = (w.packed ^ 0x88).view(torch.int32).view(2, 2, 32, 4)  # [tile, block, lane, word]
        want = torch.zeros_like(words, dtype=torch.int64)
        want[tile, block, 4 * g + t, j] = 13 << (4 * (4 * e + 2 * p + h))
        assert torch.equal(words.long() & 0xFFFFFFFF, want)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_int4_error(symmetric, group):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(24, 264, generator=g)
    w[3] = 0.0
    w[4, :32] = 0.5  # one sign: the range is widened to hold zero
    q = quantize_int4(w, group, symmetric)
    back = dequantize_int4(q)
    for j0 in range(0, 264, group):
        part = w[:, j0:j0 + group]
        if symmetric:
            step = part.abs().amax(1) / 7.0
        else:
            step = (part.amax(1).clamp(min=0) - part.amin(1).clamp(max=0)) / 15.0
        # half a step from the code's rounding, one more for the zero point's, 15 roundings of the bf16 scale
        bound = step * (0.5 if symmetric else 1.0) * (1 + 2 ** -8) + step * 15 * 2 ** -8 + 1e-12
        assert ((back[:, j0:j0 + group] - part).abs() <= bound[:, None]).all()
    assert torch.equal(back[3], torch.zeros(264))


def test_int4_linear_cpu():
    codes, scales, z, w = _weight(37, 200, 64, True, seed=5)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(5, 200, generator=g).to(torch.bfloat16)
    bias = torch.randn(37, generator=g).to(torch.bfloat16)
    want = x.double() @ dequantize_int4(w, torch.float64).t() + bias.double()
    got = ops.int4_linear(x, w, bias, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    room = (x.double().abs() @ dequantize_int4(w, torch.float64).abs().t() + bias.double().abs()) * 202 * 2 ** -24
    assert ((got.double() - want).abs() <= room).all()
    out = torch.empty(5, 37, dtype=torch.bfloat16)
    assert ops.int4_linear(x, w, bias, out=out) is out
    assert torch.equal(out, got.to(torch.bfloat16))


def test_mx8_format():
    """Every rule of the format by hand."""
    y = torch.zeros(9, 32, dtype=torch.float64)
    y[0, :4] = torch.tensor([448.0, -1.0, 17.0, 19.0])   # scale 1; 17 and 19 are ties between 16, 18 and 20
    y[1, 0] = 448.0000001                                  # just above: the next scale
    y[2, 0], y[2, 1] = 1.75 * 2.0 ** -118, 2.0 ** -120      # the smallest scale, 2^-126
    y[3, 0] = 2.0 ** -140                                   # below it: elements lose bits
    y[4, 3] = float("inf")
    y[5, 3] = float("nan")
    y[6, 3] = 1e39                                          # beyond float32
    y[7, 0], y[7, 1] = 256.0, 2.0 ** -10                    # half of E4M3's smallest step: a tie to zero
    q, sf = quantize_mx8_rows_reference(y)
    assert sf.view(-1).tolist() == [127, 128, 1, 1, 255, 255, 255, 127, 0]
    v = q.view(torch.float8_e4m3fn).float()
    assert v[0, :4].tolist() == [448.0, -1.0, 16.0, 20.0]
    assert v[1, 0] == 224.0
    assert v[2, :2].tolist() == [448.0, 64.0]
    assert v[3, 0] == 0.0
    assert v[4].isnan().all() and v[5].isnan().all() and v[6].isnan().all()
    assert v[7, :2].tolist() == [256.0, 0.0]
    assert torch.equal(q[8], torch.zeros(32, dtype=torch.uint8))
    back = dequantize_mx8_rows(q, sf)
    assert back[4].isnan().all() and back[0, 0] == 448.0 and back[8].abs().max() == 0


def test_rmsnorm_mx8_cpu():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 96, generator=g).to(torch.bfloat16)
    res = torch.randn(6, 96, generator=g).to(torch.bfloat16)
    w = torch.randn(96, generator=g).to(torch.bfloat16)
    x[2], res[2] = 0, 0
    keep = res.clone()
    q, sf = ops.rmsnorm_mx8(x, w, 1e-6, residual=res)
    assert torch.equal(res, (x.float() + keep.float()).to(torch.bfloat16))  # in place
    other = torch.empty_like(res)
    q2, sf2 = ops.rmsnorm_mx8(x, w, 1e-6, residual=keep, residual_out=other)
    assert torch.equal(other, res) and torch.equal(q, q2) and torch.equal(sf, sf2)
    q3, sf3 = ops.rmsnorm_mx8(res, w, 1e-6)
    assert torch.equal(q, q3) and torch.equal(sf, sf3)
    assert sf[2].tolist() == [0, 0, 0] and q[2].max() == 0
    v = res.double()
    want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    # E4M3: half a step of 2^-4 of the value, or of the smallest step 2^-9 under a scale of at most amax / 224
    room = want.abs() * 2 ** -4 + (want.view(6, 3, 32).abs().amax(-1) / 224 * 2 ** -10).repeat_interleave(32, 1)
    assert ((dequantize_mx8_rows(q, sf, torch.float64) - want).abs() <= room).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_act_mx8_cpu(act):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 256, generator=g) * 3
    fn = ops.silu_and_mul_mx8 if act == "silu" else ops.gelu_and_mul_mx8
    q, sf = fn(x)
    gate, up = x[:, :128].double(), x[:, 128:].double()
    y = (gate / (1 + torch.exp(-gate)) if act == "silu" else 0.5 * gate * (1 + torch.erf(gate / math.sqrt(2)))) * up
    room = y.abs() * (2 ** -4 + 1e-9) + (y.view(5, 4, 32).abs().amax(-1) / 224 * 2 ** -10).repeat_interleave(32, 1)
    assert ((dequantize_mx8_rows(q, sf, torch.float64) - y).abs() <= room).all()
    if act == "silu":
        inter = torch.stack([x[:, :128].view(5, 2, 64), x[:, 128:].view(5, 2, 64)], dim=2).reshape(5, 256)
        q2, sf2 = ops.silu_and_mul_mx8(inter, interleaved=True)
        assert torch.equal(q, q2) and torch.equal(sf, sf2)


def test_quantised_mlp_cpu():
    """The operators as they are used together, against float64."""
    g = torch.Generator().manual_seed(9)
    h, d, T = 128, 192, 7
    x, res = (torch.randn(T, h, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(h, dtype=torch.bfloat16)
    up, down = (quantize_int4(torch.randn(*s, generator=g) * 0.1, 64) for s in [(2 * d, h), (h, d)])
    q, sf = ops.rmsnorm_mx8(x, w, 1e-6, residual=res)
    gu = ops.int4_linear(q, up, x_scales=sf)
    a, asf = ops.silu_and_mul_mx8(gu)
    y = ops.int4_linear(a, down, x_scales=asf)
    xd = dequantize_mx8_rows(q, sf, torch.float64)
    gud = xd @ dequantize_int4(up, torch.float64).t()
    assert ((gu.double() - gud).abs() <= gud.abs() * 2 ** -8 + 1e-4).all()
    yd = dequantize_mx8_rows(a, asf, torch.float64) @ dequantize_int4(down, torch.float64).t()
    assert y.dtype == torch.bfloat16 and ((y.double() - yd).abs() <= yd.abs() * 2 ** -8 + 1e-4).all()


def test_refusals():
    u8 = torch.uint8
    codes, scales = torch.zeros(4, 32, dtype=u8), torch.ones(4, 1, dtype=torch.bfloat16)
    w = int4_weight(codes, scales, None, 64)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        int4_weight(codes, scales, None, 48)                      # group
    with pytest.raises(ValueError):
        int4_weight(codes, scales.repeat(1, 2), None, 64)         # groups
    with pytest.raises(ValueError):
        int4_weight(codes, scales.float(), None, 64)              # scale type
    with pytest.raises(ValueError):
        int4_weight(codes, scales, torch.full((4, 1), 16, dtype=u8), 64)  # zero point
    with pytest.raises(ValueError):
        int4_weight(codes[:, :3], scales, None, 64)               # K = 6
    with pytest.raises(ValueError):
        int4_weight(codes.int(), scales, None, 64)
    with pytest.raises(ValueError):
        quantize_int4(torch.zeros(4, 60), 64)
    with pytest.raises(ValueError):
        ops.int4_linear(x[:, :32], w)
    with pytest.raises(ValueError):
        ops.int4_linear(x.to(u8), w)                              # no scales
    with pytest.raises(ValueError):
        ops.int4_linear(x, w, x_scales=torch.zeros(2, 2, dtype=u8))
    with pytest.raises(ValueError):
        ops.int4_linear(x, w, out=torch.zeros(2, 4), out_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.rmsnorm_mx8(torch.zeros(2, 48), None, 1e-6)
    with pytest.raises(ValueError):
        ops.rmsnorm_mx8(torch.zeros(2, 64), None, 1e-6, residual_out=torch.zeros(2, 64))
    with pytest.raises(ValueError):
        ops.silu_and_mul_mx8(torch.zeros(2, 96))
    with pytest.raises(ValueError):
        ops.silu_and_mul_mx8(torch.zeros(2, 64), interleaved=True)
    with pytest.raises(RuntimeError):
        ops.silu_and_mul_mx8(torch.zeros(2, 128), out=(torch.zeros(2, 64), torch.zeros(2, 2)))
    with pytest.raises(ValueError):
        quantize_mx8_rows_reference(torch.zeros(2, 40))


def test_native_messages_with_numbers():
    """A refusal whose message holds numbers raises (formatting them must not crash the process)."""
    if not ops.native_available():
        pytest.skip("native library not built")
    t = torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="group of 32, 64 or 128, got 48"):
        ops.native().Int4Handle(t, t, None, t, 4, 64, 48, t)
    with pytest.raises(RuntimeError, match=r"got \[4, 60\]"):
        ops.native().Int4Handle(t, t, None, t, 4, 60, 64, t)
    with pytest.raises(RuntimeError, match="codes of the wrong type, size or alignment"):
        ops.native().Int4Handle(t, t, None, t, 4, 64, 64, t)  # on the CPU


def test_weight_parts_are_not_replaced():
    w = quantize_int4(torch.randn(32, 64), 64)
    with pytest.raises(AttributeError):
        w.packed = w.packed.clone()
