"""4-bit linear, RMSNorm and gated activations with MXFP8 output on the GPU,
against float64 (the MXFP8 bits exactly: the kernels round at the borders as
64 bits do; the products within the rounding of their sums and output)."""

import pytest
import torch

from minisgl import ops
from minisgl.ops import reference as ref
from minisgl.quant import dequantize_int4, dequantize_mx8_rows, int4_weight, quantize_int4
from minisgl.quant.int4 import _pack_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _same_rows(got, want):
    q, sf = got
    wq, wsf = want
    assert torch.equal(sf, wsf), (sf != wsf).nonzero()[:8].tolist()
    bad = q != wq
    assert not bool(bad.any()), (bad.nonzero()[:8].tolist(), q[bad][:8].tolist(), wq[bad][:8].tolist())


# ------------------------------------------------------------------ RMSNorm
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (2, 1024), (5, 4128), (257, 512), (1, 5120), (4, 7168)])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("residual", ["none", "in place", "out"])
def test_rmsnorm_mx8(rows, cols, dt, residual):
    g = _gen(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * 2).to(TYPES[dt])
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(TYPES[dt])
    res = (torch.randn(rows, cols, generator=g, device=DEV) * 5).to(TYPES[dt]) if residual != "none" else None
    want_res = None if res is None else torch.empty_like(res)
    want = ref.rmsnorm_mx8(x, w, 1e-6, res, want_res)
    if residual == "none":
        got = ops.rmsnorm_mx8(x, w, 1e-6)
    elif residual == "in place":
        got = ops.rmsnorm_mx8(x, w, 1e-6, residual=res)
        assert torch.equal(res, want_res)
    else:
        keep, out = res.clone(), torch.empty_like(res)
        got = ops.rmsnorm_mx8(x, w, 1e-6, residual=res, residual_out=out)
        assert torch.equal(out, want_res) and torch.equal(res, keep)
    _same_rows(got, want)


@pytest.mark.parametrize("dt,cols", [("bf16", 32768), ("fp16", 16416), ("fp32", 16384)])
def test_rmsnorm_mx8_widest(dt, cols):
    x = torch.randn(3, cols, generator=_gen(cols), device=DEV).to(TYPES[dt])
    _same_rows(ops.rmsnorm_mx8(x, None, 1e-5), ref.rmsnorm_mx8(x, None, 1e-5, None, None))


# CTAs that walk several rows, the next one's copies under way while a row is written back in place: rows of one warp
# and of odd widths, either number of vectors a thread, the widest with a residual
@pytest.mark.parametrize("rows,cols,dt", [(9001, 96, "bf16"), (3001, 1056, "fp16"), (1501, 5120, "fp32"),
                                          (1201, 6272, "bf16"), (1201, 6272, "fp16"), (700, 16384, "fp32"),
                                          (600, 32768, "bf16")])
def test_rmsnorm_mx8_many_rows(rows, cols, dt):
    g = _gen(rows)
    t = TYPES[dt]
    x = torch.randn(rows, cols, generator=g, device=DEV).to(t)
    x[rows // 2] = 0
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(t)
    res = (torch.randn(rows, cols, generator=g, device=DEV) * 3).to(t)
    res[rows // 2] = 0
    want_res = torch.empty_like(res)
    want = ref.rmsnorm_mx8(x, w, 1e-6, res, want_res)
    got = ops.rmsnorm_mx8(x, w, 1e-6, residual=res)
    assert torch.equal(res, want_res)
    _same_rows(got, want)
    _same_rows(ops.rmsnorm_mx8(x, w, 1e-6), ref.rmsnorm_mx8(x, w, 1e-6, None, None))


@pytest.mark.parametrize("dt", list(TYPES))
def test_rmsnorm_mx8_hard_rows(dt):
    """Zero rows, infinities and NaN, values at the ends of the type, blocks of
    zero weight, values that lie on rounding borders, eps = 0."""
    t = TYPES[dt]
    x = torch.randn(12, 256, generator=_gen(1), device=DEV)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 200] = float("nan")
    x[3] *= torch.finfo(t).tiny * 4
    x[4] *= 1e4
    x[5] = torch.where(x[5] > 0, 1.0, -1.0)  # rms 1: y is w exactly (eps = 0)
    x[6, 32:64] *= 1e-7
    x[7] = 0
    x[7, 3] = 2.0
    x[8, :64] = 0
    x[9] = -0.0
    x[10] *= 1e-3
    x = x.to(t)
    w = torch.ones(256, device=DEV)
    w[64:96] = 0
    w[96:104] = torch.tensor([1.0625, 1.1875, 448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 464.0])
    w = w.to(t)
    for eps in (0.0, 1e-6):
        _same_rows(ops.rmsnorm_mx8(x, w, eps), ref.rmsnorm_mx8(x, w, eps, None, None))
        out = torch.empty_like(x)
        want = torch.empty_like(x)
        res = x.flip(0).contiguous()
        got = ops.rmsnorm_mx8(x, w, eps, residual=res, residual_out=out)
        _same_rows(got, ref.rmsnorm_mx8(x, w, eps, res, want))
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))
    if dt == "fp32":
        big = torch.randn(4, 256, generator=_gen(2), device=DEV) * torch.tensor([[1e30], [1e-30], [3e37], [1e-38]], device=DEV)
        for eps in (0.0, 1e-6):
            _same_rows(ops.rmsnorm_mx8(big, None, eps), ref.rmsnorm_mx8(big, None, eps, None, None))


def test_rows_on_borders_in_bulk():
    """Eight million values each: some hundred lie closer to a border than float32 can tell."""
    g = _gen(11)
    x = torch.randn(2048, 4096, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(4096, generator=g, device=DEV).to(torch.bfloat16)
    _same_rows(ops.rmsnorm_mx8(x, w, 1e-6), ref.rmsnorm_mx8(x, w, 1e-6, None, None))
    gu = (torch.randn(1024, 16384, generator=g, device=DEV) * 4).to(torch.float16)
    _same_rows(ops.silu_and_mul_mx8(gu), ref.act_mx8(gu, "silu", False))
    _same_rows(ops.gelu_and_mul_mx8(gu), ref.act_mx8(gu, "gelu", False))
    gu = torch.randn(512, 16384, generator=g, device=DEV) * 2
    _same_rows(ops.silu_and_mul_mx8(gu, interleaved=True), ref.act_mx8(gu, "silu", True))


# -------------------------------------------------------------- activations
@pytest.mark.parametrize("rows,d", [(1, 32), (3, 96), (7, 4160), (130, 64), (2, 25600)])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_act_mx8(rows, d, dt, act):
    x = (torch.randn(rows, 2 * d, generator=_gen(rows + d), device=DEV) * 3).to(TYPES[dt])
    fn = ops.silu_and_mul_mx8 if act == "silu" else ops.gelu_and_mul_mx8
    _same_rows(fn(x), ref.act_mx8(x, act, False))
    if act == "silu" and d % 64 == 0:
        _same_rows(fn(x, interleaved=True), ref.act_mx8(x, act, True))


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_act_mx8_hard_values(dt, act):
    t = TYPES[dt]
    x = torch.randn(14, 128, generator=_gen(4), device=DEV)
    g, u = x[:, :64], x[:, 64:]
    g[0] = 0
    u[1] = 0
    g[2, 3] = float("inf")
    g[3, 3] = float("-inf")
    u[4, 3] = float("nan")
    g[5] = -20.0 - 30 * g[5].abs()     # a block that is all tail
    g[6] = -100.0 - 30 * g[6].abs()    # below float32 for e^g
    g[7, ::2] = -18.0                  # tail beside ordinary values
    g[8] *= 60
    u[9] *= 6e4
    g[10] *= 1e-6
    u[10] *= 1e-6
    g[11], u[11] = 300.0, 300.0
    g[12] = -0.0
    u[13] *= torch.finfo(t).tiny
    x = x.to(t)
    fn = ops.silu_and_mul_mx8 if act == "silu" else ops.gelu_and_mul_mx8
    _same_rows(fn(x), ref.act_mx8(x, act, False))
    if dt != "fp16":
        x = torch.randn(3, 128, generator=_gen(5), device=DEV)
        x[0] *= 1e25   # products beyond float32
        x[1] *= 1e-25  # and below it
        x[2, 64:] *= 1e-30
        _same_rows(fn(x.to(t)), ref.act_mx8(x.to(t), act, False))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_act_mx8_gate_tails(dt, act):
    """Gates far below zero beside vast products: what they leave may decide a block's scale."""
    g = torch.empty(4096, 64, device=DEV).uniform_(-110, -4, generator=_gen(21))
    g[::2] = g[::2, :1]  # half of the rows: one gate a row
    u = torch.randn(4096, 64, generator=_gen(22), device=DEV)
    u *= 10.0 ** torch.empty(4096, 1, device=DEV).uniform_(-3, 37, generator=_gen(23))
    u[:, ::8] *= 10.0 ** torch.empty(4096, 1, device=DEV).uniform_(-30, 0, generator=_gen(24))
    g[3::4, 1::2] = torch.randn(1024, 32, generator=_gen(25), device=DEV)  # ordinary values beside them
    u[3::4, 1::2] = torch.randn(1024, 32, generator=_gen(26), device=DEV)
    x = torch.cat([g, u], dim=1).to(TYPES[dt])
    fn = ops.silu_and_mul_mx8 if act == "silu" else ops.gelu_and_mul_mx8
    _same_rows(fn(x), ref.act_mx8(x, act, False))


def test_rows_strided_and_given_out():
    g = _gen(8)
    base = torch.randn(9, 1024, generator=g, device=DEV).to(torch.bfloat16)
    x = base[:, 64:576]  # 512 columns of a wider row
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    q_all = torch.full((11, 640), 0xAB, dtype=torch.uint8, device=DEV)
    s_all = torch.full((11, 20), 0xCD, dtype=torch.uint8, device=DEV)
    out = (q_all[1:10, 64:576], s_all[1:10, 2:18])
    got = ops.rmsnorm_mx8(x, w, 1e-6, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    _same_rows(out, ref.rmsnorm_mx8(x, w, 1e-6, None, None))
    _same_rows(ops.silu_and_mul_mx8(x, out=(q_all[1:10, 64:320], s_all[1:10, 2:10])), ref.act_mx8(x, "silu", False))
    # what lies around the outputs stays as it was
    assert bool((q_all[0] == 0xAB).all()) and bool((q_all[10] == 0xAB).all()) and bool((q_all[:, :64] == 0xAB).all())
    assert bool((s_all[:, :2] == 0xCD).all()) and bool((s_all[:, 18:] == 0xCD).all()) and bool((s_all[10] == 0xCD).all())
    empty = ops.rmsnorm_mx8(x[:0], w, 1e-6)
    assert empty[0].shape == (0, 512) and empty[1].shape == (0, 16)
    assert ops.silu_and_mul_mx8(x[:0])[0].shape == (0, 256)


# -------------------------------------------------------------- 4-bit linear
def _weight(n, k, group, zeros, seed, dtype):
    g = _gen(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.rand(n, -(-k // group), generator=g, device=DEV) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return int4_weight(codes, scales, z, group)


def _check_linear(y, xd, w, bias, rounded=False):
    """Against float64. Every product code * x is exact; at most (16 + 1) * 4 roundings inside a block of 64
    columns, one per block and some twenty where partial sums meet (2^-23 each: a tensor core may truncate),
    then the output's half step. ``rounded``: more than 8 rows, whose product takes weights that are rounded once to
    x's 16-bit type (half a step: 2^-8 of each for bf16, less for fp16)."""
    wd = dequantize_int4(w, torch.float64)
    want = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    half = torch.finfo(y.dtype).eps / 2
    room = size * (68 + w.k / 64 + 20) * 2 ** -23 + want.abs() * half + torch.finfo(y.dtype).tiny
    if rounded:
        room = room + size * 2 ** -8
    err = (y.double() - want).abs()
    assert bool((err <= room).all()), (err / room).max().item()


@pytest.mark.parametrize("n,k", [(1, 8), (16, 64), (17, 72), (100, 1096), (33, 256), (2048, 1024)])
def test_int4_pack(n, k):
    """The kernel's layout against its statement; rows of a wider tensor too."""
    codes = torch.randint(0, 256, (n, k // 2), generator=_gen(n), device=DEV, dtype=torch.uint8)
    want = _pack_reference(codes.cpu())
    assert torch.equal(ops.native().int4_pack(codes).cpu(), want)
    wide = torch.full((n, k // 2 + 24), 0x5A, device=DEV, dtype=torch.uint8)
    wide[:, 3:3 + k // 2] = codes
    assert torch.equal(ops.native().int4_pack(wide[:, 3:3 + k // 2]).cpu(), want)


SHAPES = [(1, 16, 64), (1, 2048, 1024), (3, 17, 8), (8, 33, 72), (9, 128, 4168), (16, 1000, 512), (17, 256, 640),
          (31, 80, 1000), (32, 512, 2048), (33, 144, 320), (70, 272, 1096), (257, 384, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dt,zeros,bias", [("bf16", False, False), ("fp16", True, True), ("bf16", True, True)])
def test_int4_linear(m, n, k, group, dt, zeros, bias):
    t = TYPES[dt]
    w = _weight(n, k, group, zeros, m + n + k, t)
    g = _gen(m)
    x = torch.randn(m, k, generator=g, device=DEV).to(t)
    b = torch.randn(n, generator=g, device=DEV).to(t) if bias else None
    y = ops.int4_linear(x, w, b)
    assert y.dtype == t and y.shape == (m, n)
    _check_linear(y, x.double(), w, b, rounded=m > 8)
    _check_linear(ops.int4_linear(x, w, b, out_dtype=torch.float32), x.double(), w, b, rounded=m > 8)
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("m,n,k", [(1, 64, 32), (2, 100, 96), (8, 512, 1024), (20, 300, 2080), (40, 128, 512)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_linear_mx8_rows(m, n, k, group):
    w = _weight(n, k, group, group == 64, n, torch.bfloat16)
    x = torch.randn(m, k, generator=_gen(k), device=DEV)
    x[0, :32] *= 1e-20
    if m > 1:
        x[1] = 0
    q, sf = ops.rmsnorm_mx8(x, None, 0.0 if m == 1 else 1e-6)
    xd = dequantize_mx8_rows(q, sf, torch.float64)
    _check_linear(ops.int4_linear(q, w, x_scales=sf), xd, w, None, rounded=m > 8)
    _check_linear(ops.int4_linear(q, w, x_scales=sf, out_dtype=torch.float32), xd, w, None, rounded=m > 8)
    ops.check_device_errors(torch.device(DEV))


def test_int4_linear_mixed_types_strides_and_out():
    w = _weight(200, 256, 64, True, 3, torch.float16)  # fp16 scales under bf16 rows
    g = _gen(3)
    for m in (5, 40):
        base = torch.randn(m, 512, generator=g, device=DEV).to(torch.bfloat16)
        x = base[:, 128:384]
        bias = torch.randn(200, generator=g, device=DEV)
        wide = torch.full((m + 2, 264), 7.0, device=DEV, dtype=torch.float16)
        out = wide[1:m + 1, 8:208]
        assert ops.int4_linear(x, w, bias, out=out) is out
        _check_linear(out, x.double(), w, bias, rounded=m > 8)
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[1:m + 1, 8:208] = False
        assert bool((wide[keep] == 7.0).all())
        odd = torch.full((m + 2, 203), 7.0, device=DEV, dtype=torch.bfloat16)[1:m + 1, 1:201]
        _check_linear(ops.int4_linear(x, w, bias, out=odd), x.double(), w, bias, rounded=m > 8)
        xs = torch.randn(256, generator=g, device=DEV).to(torch.bfloat16).expand(m, 256)
        with pytest.raises(RuntimeError):
            ops.int4_linear(xs, w)  # rows that lie on one another
    assert ops.int4_linear(x[:0], w).shape == (0, 200)


@pytest.mark.parametrize("m", [1, 8, 40])
def test_int4_linear_not_finite(m):
    """An infinity or NaN of x reaches its own row alone."""
    w = _weight(64, 256, 128, False, 5, torch.bfloat16)
    x = torch.randn(m, 256, generator=_gen(5), device=DEV).to(torch.bfloat16)
    x[m - 1, 17] = float("nan")
    y = ops.int4_linear(x, w)
    assert y[m - 1].isnan().all() and y[: m - 1].isfinite().all()
    x[m - 1, 17] = float("inf")
    y = ops.int4_linear(x, w)
    want = x.float() @ dequantize_int4(w).t()
    assert torch.equal(y[m - 1].isnan(), want[m - 1].isnan()) and y[: m - 1].isfinite().all()
    assert torch.equal(y[m - 1].isinf(), want[m - 1].isinf())


# ------------------------------------------------------------------ together
def _mlp(x, res, w, up, down):
    q, sf = ops.rmsnorm_mx8(x, w, 1e-6, residual=res)
    gu = ops.int4_linear(q, up, x_scales=sf)
    a, asf = ops.silu_and_mul_mx8(gu)
    return q, sf, gu, a, asf, ops.int4_linear(a, down, x_scales=asf)


@pytest.mark.parametrize("T", [1, 6, 50])
def test_quantised_mlp(T):
    g = _gen(T)
    h, d = 512, 1024
    x, res = (torch.randn(T, h, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(h, device=DEV, dtype=torch.bfloat16)
    up, down = (quantize_int4(torch.randn(*s, generator=g, device=DEV) * 0.05, 128) for s in [(2 * d, h), (h, d)])
    start = res.clone()
    q, sf, gu, a, asf, y = _mlp(x, res, w, up, down)
    want_res = torch.empty_like(res)
    _same_rows((q, sf), ref.rmsnorm_mx8(x, w, 1e-6, start, want_res))
    assert torch.equal(res, want_res)
    _check_linear(gu, dequantize_mx8_rows(q, sf, torch.float64), up, None, rounded=T > 8)
    _same_rows((a, asf), ref.act_mx8(gu, "silu", False))
    _check_linear(y, dequantize_mx8_rows(a, asf, torch.float64), down, None, rounded=T > 8)


@pytest.mark.parametrize("T", [2, 40])
def test_captured_graphs_beside_one_another(T):
    """Two graphs of the same operators, replayed at the same time on two streams, with new inputs each time."""
    h, d = 512, 768
    g = _gen(20)
    w = torch.ones(h, device=DEV, dtype=torch.bfloat16)
    up, down = (quantize_int4(torch.randn(*s, generator=g, device=DEV) * 0.05, 64) for s in [(2 * d, h), (h, d)])
    sides = []
    for _ in range(2):
        st = torch.cuda.Stream()
        x, res = (torch.randn(T, h, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        x0, r0 = x.clone(), res.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            _mlp(x, res, w, up, down)  # warm-up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            res.copy_(r0)
            out = _mlp(x, res, w, up, down)
        sides.append((st, graph, x, x0, r0, out))
    for turn in range(3):
        want = []
        for st, graph, x, x0, r0, out in sides:
            x.copy_(x0 * (turn + 1))
            r = r0.clone()
            want.append([t.clone() for t in _mlp(x, r, w, up, down)])
        torch.cuda.synchronize()
        for _ in range(4):
            for st, graph, *_ in sides:
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for side, ws in zip(sides, want):
            for a, b in zip(side[5], ws):
                assert torch.equal(a, b)
    ops.check_device_errors(torch.device(DEV))


def test_calls_on_two_streams_at_once():
    g = _gen(30)
    w = quantize_int4(torch.randn(4096, 2048, generator=g, device=DEV) * 0.05, 128)
    xs = [torch.randn(m, 2048, generator=g, device=DEV).to(torch.bfloat16) for m in (1, 7, 24, 64)]
    want = [ops.int4_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(10):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(ops.int4_linear(x, w))
    torch.cuda.synchronize()
    for i, many in enumerate(got):
        assert all(torch.equal(y, want[i]) for y in many)  # the same bits every time
    ops.check_device_errors(torch.device(DEV))


def test_weight_made_just_before_the_call():
    """A weight that was written by the kernels right before the product that reads it."""
    g = _gen(40)
    x = torch.randn(4, 1024, generator=g, device=DEV).to(torch.bfloat16)
    for i in range(5):
        w = quantize_int4(torch.randn(1024, 1024, generator=g, device=DEV), 128)
        w2 = int4_weight(torch.zeros(1024, 512, device=DEV, dtype=torch.uint8), torch.ones(1024, 8, device=DEV, dtype=torch.bfloat16))
        w2.packed.copy_(w.packed)
        w2.scales.copy_(w.scales)
        y2 = ops.int4_linear(x, w2)
        _check_linear(y2, x.double(), w, None)


def test_refusals_gpu():
    w = _weight(32, 64, 64, False, 1, torch.bfloat16)
    x = torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x.float(), w)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w.to("cpu"))
    with pytest.raises(RuntimeError, match=r"x must be \[M, 64\], got \[2, 32\]"):
        ops.int4_linear(x[:, :32], w)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w, out=torch.zeros(2, 32, device=DEV), out_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x.to(torch.uint8), w)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w, x_scales=torch.zeros(2, 2, device=DEV, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(x[:, :48].contiguous(), None, 1e-6)
    with pytest.raises(RuntimeError):
        ops.silu_and_mul_mx8(x, interleaved=True)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w, torch.zeros(31, device=DEV))
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w, torch.zeros(32))
    with pytest.raises(RuntimeError):
        ops.int4_linear(x, w, out=torch.zeros(3, 32, device=DEV))
    with pytest.raises(RuntimeError):
        ops.int4_linear(torch.zeros(2, 66, device=DEV, dtype=torch.bfloat16)[:, 1:65], w)  # rows off 16 bytes
    with pytest.raises(RuntimeError):
        ops.int4_linear(torch.zeros(2, 64, device=DEV, dtype=torch.uint8), w, x_scales=torch.zeros(2, 1, device=DEV, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(x, torch.zeros(64, device=DEV), 1e-6)                                # another type
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(x, None, 1e-6, residual=torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(x, None, -1.0)
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(torch.zeros(1, 32800, device=DEV, dtype=torch.bfloat16), None, 1e-6)
    with pytest.raises(RuntimeError):
        ops.rmsnorm_mx8(x.int(), None, 1e-6)
    with pytest.raises(RuntimeError):
        ops.silu_and_mul_mx8(x, out=(torch.zeros(2, 32, device=DEV), torch.zeros(2, 1, device=DEV)))
    with pytest.raises(RuntimeError):
        ops.silu_and_mul_mx8(x, out=(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)))


@pytest.mark.parametrize("m,n,k,dt", [(600, 20000, 256, "bf16"), (300, 33000, 128, "fp16"), (40, 40000, 384, "bf16"), (1100, 9000, 640, "bf16")])
def test_int4_linear_many_tiles(m, n, k, dt):
    """More tiles than SMs: a CTA takes several, one after another."""
    t = TYPES[dt]
    w = _weight(n, k, 64, True, n, t)
    x = torch.randn(m, k, generator=_gen(m), device=DEV).to(t)
    _check_linear(ops.int4_linear(x, w), x.double(), w, None, rounded=True)
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("m,k", [(8, 40000), (3, 100000), (1, 300000)])
@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_int4_linear_few_rows_too_wide_to_stream(m, k, kind):
    """Rows that shared memory cannot hold take the tiles of the longer batches."""
    w = _weight(48, k, 128, True, m, torch.bfloat16)
    x = torch.randn(m, k, generator=_gen(k), device=DEV)
    if kind == "mx8":
        q = torch.randint(0, 0x7E, (m, k), generator=_gen(k), device=DEV, dtype=torch.uint8)
        sf = torch.randint(118, 124, (m, k // 32), generator=_gen(m), device=DEV, dtype=torch.uint8)
        _check_linear(ops.int4_linear(q, w, x_scales=sf), dequantize_mx8_rows(q, sf, torch.float64), w, None, rounded=True)
    else:
        x = x.to(torch.bfloat16)
        _check_linear(ops.int4_linear(x, w), x.double(), w, None, rounded=True)
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("m", [2, 12])
def test_int4_linear_wide_range_of_x(m):
    """Magnitudes from one end of bf16 to the other, in columns of their own and beside one another; every group
    has weights other than its zero point under its largest x, so the sum is as large as its terms."""
    w = _weight(64, 1024, 64, False, 2, torch.bfloat16)
    x = torch.randn(m, 1024, generator=_gen(9), device=DEV)
    x[:, :128] *= 1e30
    x[:, 128:256] *= 1e-30
    x[:, 256:384] *= torch.logspace(-20, 20, 128, device=DEV)
    x[0] *= 1e-5
    x = x.to(torch.bfloat16)
    y = ops.int4_linear(x, w, out_dtype=torch.float32)
    wd = dequantize_int4(w, torch.float64)
    want, size = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    # x's integers: at most half a unit off each. The unit is 2^-21 of the largest value's power of two, but never
    # below 2^-122, because its inverse is a float32 factor (2^122) and the factor that undoes it and the codes'
    # sixteenths, 2^-126, has to be normal.
    def half_units(z, weights):
        top = z.double().abs().view(m, -1, 128).amax(-1)
        return torch.einsum("mb,nb->mn", (top * 2 ** -22).clamp(min=2.0 ** -123), weights.abs().view(64, -1, 128).sum(-1))

    fixed = half_units(x, wd)
    room = size * (68 + 1024 / 64 + 20) * 2 ** -23 + want.abs() * 2 ** -24 + (fixed if m <= 8 else size * 2 ** -8)
    assert bool(((y.double() - want).abs() <= room).all())
    if m <= 8:  # tiny and huge alone
        for cols in (slice(0, 128), slice(128, 256)):
            z = torch.zeros_like(x)
            z[:, cols] = x[:, cols]
            got, ref_ = ops.int4_linear(z, w, out_dtype=torch.float32).double(), z.double() @ wd.t()
            s = z.double().abs() @ wd.abs().t()
            assert bool(((got - ref_).abs() <= s * 104 * 2 ** -23 + half_units(z[:, cols], wd[:, cols]) + 1e-45).all())


def test_int4_linear_nan_block_of_mx8():
    w = _weight(40, 256, 32, True, 6, torch.bfloat16)
    for m in (2, 20):
        q, sf = ops.rmsnorm_mx8(torch.randn(m, 256, generator=_gen(1), device=DEV), None, 1e-6)
        q[1, 32:64], sf[1, 1] = 0x7F, 255
        y = ops.int4_linear(q, w, x_scales=sf)
        assert y[1].isnan().all() and y[0].isfinite().all() and y[2:].isfinite().all()


@pytest.mark.parametrize("scale", [1e-7, 6e-5, 3e4])
def test_int4_linear_fp16_scales_at_the_ends(scale):
    """Tiny and large fp16 scales: the products of longer batches take each row's power of two out."""
    g = _gen(3)
    codes = torch.randint(0, 256, (64, 256), generator=g, device=DEV, dtype=torch.uint8)
    scales = (scale * (1 + torch.rand(64, 4, generator=g, device=DEV))).to(torch.float16)
    w = int4_weight(codes, scales, None, 128)
    for m in (4, 40):
        x = (torch.randn(m, 512, generator=g, device=DEV) * 1e-3).to(torch.float16)
        _check_linear(ops.int4_linear(x, w, out_dtype=torch.float32), x.double(), w, None, rounded=m > 8)


@pytest.mark.parametrize("m,group", [(1, 64), (7, 32), (200, 64), (30, 32)])
def test_first_call_inside_a_capture(m, group):
    """A variant's first call may be captured: nothing of its set-up is a stream operation."""
    w = _weight(704, 1152, group, True, m, torch.float16)
    x = torch.randn(m, 1152, generator=_gen(m), device=DEV).to(torch.float16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.int4_linear(x, w)
    graph.replay()
    torch.cuda.synchronize()
    _check_linear(y, x.double(), w, None, rounded=m > 8)


def test_weight_copies():
    import copy

    w = _weight(32, 128, 32, True, 1, torch.bfloat16)
    x = torch.randn(3, 128, generator=_gen(1), device=DEV).to(torch.bfloat16)
    assert torch.equal(ops.int4_linear(x, copy.deepcopy(w)), ops.int4_linear(x, w))
    assert torch.equal(ops.int4_linear(x, w.to("cpu").to(DEV)), ops.int4_linear(x, w))


# Sizes at which the estimate takes each of the few-row product's plans on 148 SMs (8 or 16 warps a CTA, one or two
# 16-row tiles a unit, a tile's columns on 1 to 8 CTAs), with rows and columns that end inside a tile
@pytest.mark.parametrize("m,n,k,group,zeros", [
    (1, 8200, 4104, 32, True), (1, 1001, 26120, 128, True),                             # 8 warps, two tiles
    (3, 4111, 2056, 64, False), (3, 1001, 8200, 32, False), (8, 333, 4104, 32, True), (8, 24, 4104, 128, False),
    (8, 6151, 520, 32, True), (3, 8200, 8200, 32, False), (8, 1001, 4104, 64, True), (8, 24, 26120, 32, False),
    (1, 8200, 8200, 32, True), (8, 20501, 4104, 128, True), (8, 10251, 4104, 32, True), (8, 6151, 8200, 128, True)])
def test_int4_linear_every_plan(m, n, k, group, zeros):
    w = _weight(n, k, group, zeros, n, torch.bfloat16)
    x = torch.randn(m, k, generator=_gen(k), device=DEV).to(torch.bfloat16)
    b = torch.randn(n, generator=_gen(n + 1), device=DEV)
    y = ops.int4_linear(x, w, b, out_dtype=torch.float32)
    _check_linear(y, x.double(), w, b)
    assert torch.equal(y, ops.int4_linear(x, w, b, out_dtype=torch.float32))  # every sum has one order
    x[0, k // 2] = float("inf")
    x[m - 1, k - 1] = float("nan")
    odd = ops.int4_linear(x, w, b, out_dtype=torch.float32)
    assert bool(odd[m - 1].isnan().all())
    if m > 2:
        assert torch.equal(odd[1], y[1]) and not bool(odd[0].isfinite().any())


@pytest.mark.parametrize("m,k", [(8, 80000), (3, 220000), (1, 700000)])
@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_int4_linear_few_rows_beyond_any_plan(m, k, kind):
    """Rows that shared memory cannot hold under any plan take the tiles of the longer batches and their scratch."""
    w = _weight(40, k, 64, True, m, torch.bfloat16)
    if kind == "mx8":
        q = torch.randint(0, 0x7E, (m, k), generator=_gen(k), device=DEV, dtype=torch.uint8)
        sf = torch.randint(118, 124, (m, k // 32), generator=_gen(m), device=DEV, dtype=torch.uint8)
        y, xd = ops.int4_linear(q, w, x_scales=sf), dequantize_mx8_rows(q, sf, torch.float64)
    else:
        x = torch.randn(m, k, generator=_gen(k), device=DEV).to(torch.bfloat16)
        y, xd = ops.int4_linear(x, w), x.double()
    _check_linear(y, xd, w, None, rounded=True)
    ops.check_device_errors(torch.device(DEV))
