"""4-bit weights whose parts are written after they were made: products that read the rows' powers of two."""

import copy
import pickle

import pytest
import torch

from minisgl import ops
from minisgl.quant import dequantize_int4, int4_weight, quantize_int4
from test_quant_tiles_gpu import _gen, _weight, check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("factor,dtype", [(1e-6, torch.bfloat16), (1e6, torch.bfloat16), (1e3, torch.float16)])
@pytest.mark.parametrize("m,k", [(40, 1032), (1, 700000)])  # the second: one row that takes the tiles
def test_scales_written_after_the_weight_was_made(m, k, factor, dtype):
    w = _weight(200 if m > 1 else 16, k, 64, True, 1, dtype)
    x = (torch.randn(m, k, generator=_gen(m), device=DEV) * 1e-2).half()
    check(ops.int4_linear(x, w, out_dtype=torch.float32), x.double(), w, None, True)
    w.scales.copy_((w.scales.float() * factor).to(dtype))
    fresh = int4_weight_like(w)
    for made in (w, w.to(DEV), copy.deepcopy(w)):
        y = ops.int4_linear(x, made, out_dtype=torch.float32)
        check(y, x.double(), fresh, None, True)
        assert torch.equal(y, ops.int4_linear(x, fresh, out_dtype=torch.float32))
    ops.check_device_errors(torch.device(DEV))


def int4_weight_like(w):
    """The same weight, made from its scales as they are."""
    from minisgl.quant import int4_codes

    def rows(t):
        return t.permute(0, 3, 2, 1).reshape(-1, t.shape[1])[: w.n, : -(-w.k // w.group)].contiguous()

    c = int4_codes(w)
    z = None if w.zeros is None else rows(torch.stack([w.zeros & 15, w.zeros >> 4], dim=-1))
    return int4_weight((c[:, 0::2] | (c[:, 1::2] << 4)).contiguous(), rows(w.scales), z, w.group)


@pytest.mark.parametrize("m", [4, 40])
def test_a_captured_product_takes_the_weight_copied_in(m):
    n, k = 200, 1032
    w = _weight(n, k, 64, True, 1, torch.float16)
    x = (torch.randn(m, k, generator=_gen(m), device=DEV) * 1e-2).half()
    ops.int4_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.int4_linear(x, w, out_dtype=torch.float32)
    for seed, factor in [(2, 1e4), (3, 1.0), (4, 1e-3)]:
        new = _weight(n, k, 64, True, seed, torch.float16)
        new.scales.copy_((new.scales.float() * factor).half())
        w.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.int4_linear(x, int4_weight_like(new), out_dtype=torch.float32))


def test_scales_written_inside_a_capture():
    w = _weight(200, 1032, 64, True, 1, torch.float16)
    x = (torch.randn(40, 1032, generator=_gen(1), device=DEV) * 1e-2).half()
    new = w.scales.clone()
    ops.int4_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.scales.copy_(new)
        y = ops.int4_linear(x, w, out_dtype=torch.float32)
    for factor in (1e4, 1e-7):
        new.mul_(factor)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.int4_linear(x, int4_weight_like(w), out_dtype=torch.float32))


@pytest.mark.parametrize("rows", [2, 40])
def test_two_graphs_replayed_beside_one_another(rows):
    """Norm, product, activation and product captured twice, each graph with tensors of its own that live as long as it
    (the residual stream among them, which the graph writes), replayed on two streams at once."""
    h, d = 512, 768
    g = _gen(20)
    norm = torch.ones(h, device=DEV, dtype=torch.bfloat16)
    up, down = (quantize_int4(torch.randn(*s, generator=g, device=DEV) * 0.05, 64) for s in [(2 * d, h), (h, d)])

    def layer(x, res):
        q, sf = ops.rmsnorm_mx8(x, norm, 1e-6, residual=res)
        a, asf = ops.silu_and_mul_mx8(ops.int4_linear(q, up, x_scales=sf))
        return q, sf, res, a, asf, ops.int4_linear(a, down, x_scales=asf)

    sides = []
    for _ in range(2):
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        x, start = (torch.randn(rows, h, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        res = start.clone()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            res.copy_(start)
            out = layer(x, res)
        sides.append((stream, graph, x, start, out))
    for turn in range(20):
        want = []
        for _, _, x, start, _ in sides:
            x.copy_(torch.randn(rows, h, generator=g, device=DEV))
            want.append([t.clone() for t in layer(x, start.clone())])
        torch.cuda.synchronize()
        for _ in range(4):
            for stream, graph, *_ in sides:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for side, ws in zip(sides, want):
            assert all(torch.equal(a, b) for a, b in zip(side[4], ws)), turn
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("how", ["to", "pickle", "copy"])
@pytest.mark.parametrize("m", [3, 40])
def test_a_weight_that_was_moved_is_ready_for_a_capture(monkeypatch, how, m):
    """The error word that its calls write to is not made inside a capture, where each replay would clear it."""
    w = _weight(200, 1032, 64, True, 1, torch.float16)
    x = (torch.randn(m, 1032, generator=_gen(1), device=DEV) * 1e-2).half()
    want = ops.int4_linear(x, w)
    ops.check_device_errors(torch.device(DEV))
    data, cpu = pickle.dumps(w), w.to("cpu")
    monkeypatch.setattr(ops, "_ERR_WORDS", {})  # as in a process that has used no kernel yet
    moved = cpu.to(DEV) if how == "to" else pickle.loads(data) if how == "pickle" else copy.deepcopy(w)
    assert len(ops._ERR_WORDS) == 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.int4_linear(x, moved)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    word = ops.error_word(torch.device(DEV))
    word[0] = 77
    graph.replay()
    assert word[0].item() == 77
    word.zero_()


# MXFP8 rows that take the tiles are widened by a kernel of their own: more than 8, or too wide to stream
@pytest.mark.parametrize("m,k,kind,launches", [(0, 1024, "bf16", 0), (8, 1024, "mx8", 1), (9, 1024, "mx8", 2),
                                               (40, 1024, "bf16", 1), (1, 700000 // 32 * 32, "mx8", 2),
                                               (1, 700000, "bf16", 1)])
def test_launches_are_counted_as_they_happen(m, k, kind, launches):
    w = _weight(32, k, 64, False, 1, torch.bfloat16)
    if kind == "mx8":
        x = torch.randint(0, 0x7E, (m, k), device=DEV, dtype=torch.uint8)
        scales = torch.full((m, k // 32), 120, device=DEV, dtype=torch.uint8)
    else:
        x, scales = torch.zeros(m, k, device=DEV, dtype=torch.bfloat16), None
    before = ops.LAUNCHES[0]
    ops.int4_linear(x, w, x_scales=scales)
    assert ops.LAUNCHES[0] - before == launches
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, 2.0 ** -25), (torch.bfloat16, 1.3e-7), (torch.float16, 2.0 ** -20),
                                       (torch.float16, 1e-5)])
@pytest.mark.parametrize("m", [8, 40])
def test_groups_far_below_a_rows_largest_scale(m, dtype, low):
    """fp16 rows that meet only the groups of small scales: the weights are as good as 16-bit weights are, whatever
    the scale of a group that x is zero under. 16-bit weights: half a step, 2^-11 of each, and the sums."""
    k = 1024
    g = _gen(1)
    codes = torch.randint(0, 256, (200, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (low * (1 + torch.rand(200, k // 64, generator=g, device=DEV))).to(dtype)
    scales[:, 3] = 1.0
    w = int4_weight(codes, scales, None, 64)
    x = torch.randn(m, k, generator=g, device=DEV).half()
    x[:, 192:256] = 0
    y = ops.int4_linear(x, w, out_dtype=torch.float32).double()
    wd, xd = dequantize_int4(w, torch.float64), x.double()
    room = xd.abs() @ wd.abs().t() * (2 ** -11 + (k // 16 * 17 + 104) * 2 ** -23)
    err = (y - xd @ wd.t()).abs()
    assert bool((err <= room).all()), (err / room).max().item()


@pytest.mark.parametrize("scale", [2.0 ** -133, 2.0 ** -126, 2.0 ** -120, 2.0 ** 89])
def test_rows_of_the_ends_of_bf16(scale):
    w = int4_weight(torch.full((40, 64), 0x99, device=DEV, dtype=torch.uint8),
                    torch.full((40, 1), scale, device=DEV, dtype=torch.bfloat16), None, 128)  # every code is 9: W = scale
    x = torch.ones(16, 128, device=DEV, dtype=torch.float16) * 2.0 ** 10
    y = ops.int4_linear(x, w, out_dtype=torch.float32)
    assert torch.equal(y, torch.full_like(y, 2.0 ** 17 * scale))


@pytest.mark.parametrize("m", [1, 8, 16])
def test_the_largest_scales(m):
    """A group's sum under the largest scale that a weight may have: 128 columns, codes 15 away from their zero point."""
    w = int4_weight(torch.full((40, 64), 0xFF, device=DEV, dtype=torch.uint8),
                    torch.full((40, 1), 2.0 ** 90, device=DEV, dtype=torch.bfloat16),
                    torch.zeros(40, 1, device=DEV, dtype=torch.uint8), 128)
    x = torch.full((m, 128), 1.9921875, device=DEV, dtype=torch.bfloat16)  # the largest below 2
    y = ops.int4_linear(x, w, out_dtype=torch.float32)
    assert torch.equal(y, torch.full_like(y, 1.9921875 * 128 * 15 * 2.0 ** 90))
