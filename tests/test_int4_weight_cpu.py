"""4-bit weights whose parts are written after they were made, on the CPU."""

import copy
import pickle

import pytest
import torch

from minisgl import ops
from minisgl.quant import Int4Weight, dequantize_int4, int4_weight, quantize_int4


def _parts(n=40, k=264, group=64, zeros=True, seed=0, factor=1.0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, -(-k // group), generator=g) * 0.02 + 0.001) * factor).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z, group


@pytest.mark.parametrize("inference", [False, True])
def test_row_powers_follow_the_scales(inference):
    with torch.inference_mode(inference):
        w = int4_weight(*_parts())
        other = int4_weight(*_parts(factor=1e3))
        assert not torch.equal(w.row_pow, other.row_pow)
        w.scales.copy_(other.scales)
        for made in (w, w.to("cpu"), copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
            assert torch.equal(made.row_pow, other.row_pow)
            assert torch.equal(made.scales, other.scales)


def test_copy_into_a_weight():
    w, new = int4_weight(*_parts()), int4_weight(*_parts(seed=1, factor=30.0))
    parts = [t.data_ptr() for t in (w.packed, w.scales, w.zeros, w.row_pow)]
    assert w.copy_(new) is w
    assert [t.data_ptr() for t in (w.packed, w.scales, w.zeros, w.row_pow)] == parts
    assert torch.equal(dequantize_int4(w), dequantize_int4(new)) and torch.equal(w.row_pow, new.row_pow)
    w.scales.mul_(2)
    new.copy_(w)  # from one whose own powers were left behind
    assert torch.equal(new.row_pow, w.row_pow) and torch.equal(new.scales, w.scales)


def test_copy_refusals():
    w = int4_weight(*_parts())
    for other in (dict(n=41), dict(n=80), dict(k=272), dict(group=32), dict(zeros=False), dict(dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            w.copy_(int4_weight(*_parts(**other)))
    with pytest.raises((ValueError, TypeError, AttributeError)):
        w.copy_(torch.zeros(3))
    assert isinstance(w, Int4Weight) and torch.equal(dequantize_int4(w), dequantize_int4(int4_weight(*_parts())))


@pytest.mark.parametrize("scale,dtype", [(2.0 ** 91, torch.bfloat16), (-(2.0 ** 91), torch.bfloat16),
                                         (float("inf"), torch.bfloat16), (float("nan"), torch.bfloat16),
                                         (float("inf"), torch.float16), (float("nan"), torch.float16)])
def test_scales_beyond_the_products_are_refused(scale, dtype):
    codes, scales, z, group = _parts(dtype=dtype)
    scales[3, 1] = 2.0 ** 90 if dtype == torch.bfloat16 else 65504.0
    int4_weight(codes, scales, z, group)
    scales[3, 1] = scale
    with pytest.raises(ValueError, match="finite"):
        int4_weight(codes, scales, z, group)


def test_weights_too_large_for_their_scales_are_refused():
    w = torch.full((4, 64), 7e5)
    quantize_int4(w, 64)
    with pytest.raises(ValueError, match="finite"):
        quantize_int4(w, 64, scale_dtype=torch.float16)  # 10^5 is beyond fp16
    with pytest.raises(ValueError, match="finite"):
        quantize_int4(w * 1e30, 64)
    w[1, 3] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        quantize_int4(w, 64)


def test_to_takes_a_device_alone():
    w = int4_weight(*_parts())
    for bad in (torch.float16, torch.zeros(1)):
        with pytest.raises((TypeError, RuntimeError)):
            w.to(bad)
    assert w.to("cpu").packed.dtype == torch.uint8 and w.to(torch.device("cpu")).n == w.n


def test_shapes_that_the_cpu_form_refuses_as_the_kernels_do():
    w = int4_weight(*_parts(n=40, k=264))
    x = torch.zeros(1, 264, dtype=torch.float16)
    for bad in (torch.zeros(3, 40, dtype=torch.float16), torch.zeros(40, dtype=torch.float16)):
        with pytest.raises(ValueError, match="out must be"):
            ops.int4_linear(x, w, out=bad)
    for bias in (torch.zeros(1), torch.zeros(39)):
        with pytest.raises(ValueError, match="bias must be"):
            ops.int4_linear(x, w, bias)
    y = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="residual"):
        ops.rmsnorm_mx8(y, None, 1e-6, residual=torch.zeros(1, 64), residual_out=torch.zeros(2, 64))
    with pytest.raises(ValueError, match="residual"):
        ops.rmsnorm_mx8(y, None, 1e-6, residual=torch.zeros(2, 64), residual_out=torch.zeros(4, 2, 64))
    with pytest.raises(ValueError, match="w must"):
        ops.rmsnorm_mx8(y, torch.ones(1), 1e-6)


@pytest.mark.parametrize("how", ["made", "copied", "pickled"])
def test_a_weight_of_inference_mode_is_copied_into_outside_of_it(how):
    with torch.inference_mode():
        w = int4_weight(*_parts())
        w = w if how == "made" else copy.deepcopy(w) if how == "copied" else pickle.loads(pickle.dumps(w))
    new = int4_weight(*_parts(seed=3, factor=40.0))
    w.copy_(new)
    w.scales.mul_(0.5)
    assert torch.equal(w.packed, new.packed) and torch.equal(w.row_pow[:40], new.row_pow[:40] * 0.5)  # padding rows keep 1
    with torch.inference_mode():
        assert torch.equal(dequantize_int4(w), dequantize_int4(new.copy_(w)))


def test_scales_of_a_parameter():
    codes, scales, z, group = _parts()
    w = int4_weight(codes, torch.nn.Parameter(scales), z, group)
    assert not w.scales.requires_grad and not w.row_pow.requires_grad
    assert w.copy_(int4_weight(*_parts(seed=5))) is w and copy.deepcopy(w).n == w.n
