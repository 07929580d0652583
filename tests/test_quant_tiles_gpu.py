"""The 4-bit product of more than 8 rows at every width of its tiles, over rings that turn many times, against the
weights rounded as the kernel rounds them; and of few rows as wide as they stream, against the weights as they are."""

import pytest
import torch

from minisgl import ops
from minisgl.quant import dequantize_int4, dequantize_mx8_rows, int4_codes, int4_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _weight(n, k, group, zeros, seed, dtype):
    g = _gen(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.rand(n, -(-k // group), generator=g, device=DEV) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return int4_weight(codes, scales, z, group)


def rounded_weight(w, half):
    """[N, K] float64: (c - z) s rounded once to bf16, or to fp16 under the row's power of two."""
    of = torch.arange(w.k, device=w.device) // w.group

    def spread(t):  # [tile, group, g, h] -> [N, K]
        return t.permute(0, 3, 2, 1).reshape(-1, t.shape[1])[: w.n].double()[:, of]

    z = 8.0 if w.zeros is None else spread(torch.stack([w.zeros & 15, w.zeros >> 4], dim=-1))
    c, s = int4_codes(w).double() - z, spread(w.scales)
    if not half:
        return (c * s).to(torch.bfloat16).double()  # 16 bits at most: exact in the float32 that torch goes through
    power = w.row_pow[: w.n, None].double()
    return (c * (s / power).half().double()).half().double() * power


def check(y, xd, w, bias, half):
    """Products of two 16-bit values are exact. A product instruction adds 16 of them to the running sum, 17 terms
    that a tensor core may each cut at 2^-23 of the largest: no larger than the running sum before a step of 128
    columns and what the step adds to it in magnitude, B (twice the sum, since a CTA of a cluster starts in the
    middle). K / 16 instructions, and 8 sums of 8 CTAs' parts; then the bias and the output's half step."""
    wd = rounded_weight(w, half)
    want = torch.zeros(xd.shape[0], w.n, dtype=torch.float64, device=DEV)
    largest, step = want.clone(), want.clone()
    for k in range(0, w.k, 128):
        xs, ws = xd[:, k:k + 128], wd[:, k:k + 128]
        want += xs @ ws.t()
        largest = torch.maximum(largest, want.abs())
        step = torch.maximum(step, xs.abs() @ ws.abs().t())
    room = (-(-w.k // 16) * 17 + 8) * 2 ** -23 * (2 * largest + step)
    if bias is not None:
        room = room + bias.double().abs() * 2 ** -23
        want = want + bias.double()
    room = room + want.abs() * (torch.finfo(y.dtype).eps / 2) + 1e-30
    err = (y.double() - want).abs()
    assert bool((err <= room).all()), ((err / room).max().item(), (err > room).nonzero()[:4].tolist())


# Rows and outputs that end inside a tile; how many clusters fit, and so where each width begins, depends on the device.
ROWS = (9, 40, 65, 100, 200, 250, 300, 384, 500)
OUTPUTS = (201, 1000, 1500, 2056, 4104, 8203, 12296, 16400, 20001)


def _size(rows, kind, k, group, half):
    """A size that the product cuts into tiles of so many rows of x: one tile to a CTA, several, or one to a cluster."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for m in ROWS:
        for n in OUTPUTS:
            got, share = ops.native().int4_tiles(m, n, k, group, half)
            several = -(-m // rows) * -(-n // 128) > sms
            if (got, share > 1, several) == (rows, kind == "cluster", kind == "several"):
                return m, n
    raise AssertionError(f"no size takes tiles of {rows} rows, {kind}")


# x comes in one copy a step where K is a multiple of 64, else in two
@pytest.mark.parametrize("rows,tiles", [(32, "one"), (32, "cluster"), (64, "one"), (64, "several"), (64, "cluster"),
                                        (128, "one"), (128, "several"), (128, "cluster"), (192, "one"),
                                        (192, "several"), (256, "one")])
@pytest.mark.parametrize("kind,group,zeros,bias,k", [("bf16", 128, False, False, 5128), ("bf16", 32, True, True, 5128),
                                                     ("fp16", 64, True, False, 5128), ("fp16", 128, False, True, 5128),
                                                     ("mx8", 64, False, False, 5152), ("bf16", 128, True, False, 5120),
                                                     ("fp16", 32, False, False, 5184), ("mx8", 128, True, True, 5120)])
def test_every_tile_width(rows, tiles, kind, group, zeros, bias, k):
    """40 or 41 steps of 128 columns: every ring turns at least six times."""
    half = kind == "fp16"
    t = torch.float16 if half else torch.bfloat16
    m, n = _size(rows, tiles, k, group, half)
    w = _weight(n, k, group, zeros, m + n, t)
    x = torch.randn(m, k, generator=_gen(m), device=DEV)
    b = torch.randn(n, generator=_gen(n), device=DEV) if bias else None
    if kind == "mx8":
        q, sf = ops.rmsnorm_mx8(x, None, 1e-6)
        call, xd = (lambda **kw: ops.int4_linear(q, w, b, x_scales=sf, **kw)), dequantize_mx8_rows(q, sf, torch.float64)
    else:
        x = x.to(t)
        call, xd = (lambda **kw: ops.int4_linear(x, w, b, **kw)), x.double()
    y = call(out_dtype=torch.float32)
    check(y, xd, w, b, half)
    assert torch.equal(call(), y.to(t))  # the same sums, stored as 16-bit values
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("m,n,k,group,kind", [(16, 1000, 4168, 32, "bf16"), (17, 256, 640, 64, "fp16"),
                                              (33, 144, 320, 128, "bf16"), (70, 272, 1096, 32, "fp16"),
                                              (31, 80, 1000, 128, "fp16"), (257, 384, 512, 64, "bf16"),
                                              (600, 20000, 256, 64, "bf16"), (300, 33000, 128, 64, "fp16"),
                                              (9, 40, 8, 32, "bf16"), (1100, 9000, 640, 64, "bf16")])
def test_other_sizes(m, n, k, group, kind):
    half = kind == "fp16"
    t = torch.float16 if half else torch.bfloat16
    w = _weight(n, k, group, True, n, t)
    x = torch.randn(m, k, generator=_gen(m), device=DEV).to(t)
    check(ops.int4_linear(x, w, out_dtype=torch.float32), x.double(), w, None, half)
    ops.check_device_errors(torch.device(DEV))


# rows of K columns beyond any plan of the few-row product (300000 in groups of 64 with zero points by 480 bytes: 293
# steps of 544 a CTA of eight, 64, a ring of 52992, 20480 for partial sums, of 232448): the tiles, over thousands of steps
@pytest.mark.parametrize("m,k", [(8, 80000), (1, 300000), (1, 700000)])
def test_few_rows_beyond_any_plan(m, k):
    w = _weight(40, k, 64, True, m, torch.bfloat16)
    x = torch.randn(m, k, generator=_gen(k), device=DEV).to(torch.bfloat16)
    check(ops.int4_linear(x, w, out_dtype=torch.float32), x.double(), w, None, False)
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("m,k,group,zeros", [(8, 40000, 128, True), (3, 100000, 32, False), (3, 100000, 128, True),
                                               (1, 300000, 128, True)])
def test_few_rows_as_wide_as_they_stream(m, k, group, zeros):
    """x as integers of half a unit's error, 2^-22 of the largest of its 128 columns at most. A group's sum comes in
    two exact integers; the lower one, up to group * 2^16 * 2^8 in sixteenths of a unit with its zero point's part, is
    rounded to 24 bits: group / 16 units of 2^-21 of the largest. Then some four roundings a group, of the group's sum
    or of the running one (starting anywhere: B as in ``check``), and forty where partial sums meet. The tiles, whose
    weights are rounded to bf16, would leave this bound."""
    w = _weight(40, k, group, zeros, m, torch.bfloat16)
    x = torch.randn(m, k, generator=_gen(k), device=DEV).to(torch.bfloat16)
    y = ops.int4_linear(x, w, out_dtype=torch.float32).double()
    wd, xd = dequantize_int4(w, torch.float64), x.double()
    scales = w.scales.permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:40].double()
    want = torch.zeros(m, 40, dtype=torch.float64, device=DEV)
    largest, step, fixed = want.clone(), want.clone(), want.clone()
    for i, c in enumerate(range(0, k, 128)):
        xs, ws = xd[:, c:c + 128], wd[:, c:c + 128]
        want += xs @ ws.t()
        largest = torch.maximum(largest, want.abs())
        step = torch.maximum(step, xs.abs() @ ws.abs().t())
        per = 128 // group
        top, s = xs.abs().amax(1)[:, None], scales[:, i * per:(i + 1) * per].sum(1)[None]
        fixed += top * (2 ** -22 * ws.abs().sum(1)[None] + group / 16 * 2 ** -21 * s)
    room = fixed + (4 * (k // group + 1) + 40) * 2 ** -24 * (2 * largest + step) + 1e-30
    err = (y - want).abs()
    assert bool((err <= room).all()), (err / room).max().item()
    rounded = xd @ rounded_weight(w, False).t()
    assert bool(((rounded - want).abs() > room).any())


@pytest.mark.parametrize("m", [5, 40])
def test_mx8_rows_of_wider_tensors(m):
    """Rows and scales that ``rmsnorm_mx8`` wrote into parts of larger tensors."""
    k, n = 1056, 200
    w = _weight(n, k, 32, True, 2, torch.bfloat16)
    q = torch.full((m + 2, k + 96), 0x7F, device=DEV, dtype=torch.uint8)[1:m + 1, 48:48 + k]
    sf = torch.full((m + 2, k // 32 + 5), 0xFF, device=DEV, dtype=torch.uint8)[1:m + 1, 3:3 + k // 32]
    ops.rmsnorm_mx8(torch.randn(m, k, generator=_gen(1), device=DEV), None, 1e-6, out=(q, sf))
    y = ops.int4_linear(q, w, x_scales=sf, out_dtype=torch.float32)
    assert torch.equal(y, ops.int4_linear(q.contiguous(), w, x_scales=sf.contiguous(), out_dtype=torch.float32))
    if m > 8:
        check(y, dequantize_mx8_rows(q, sf, torch.float64), w, None, False)
    ops.check_device_errors(torch.device(DEV))


@pytest.mark.parametrize("rows,cols", [(3, 96), (1500, 5120)])
def test_residual_sum_over_the_norms_input(rows, cols):
    """residual_out may be x itself, and x may be the residual stream too."""
    g = _gen(rows)
    x, res = (torch.randn(rows, cols, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    total = torch.empty_like(x)
    want = ops.rmsnorm_mx8(x, None, 1e-6, residual=res, residual_out=total)
    keep = x.clone()
    got = ops.rmsnorm_mx8(x, None, 1e-6, residual=res, residual_out=x)
    assert torch.equal(x, total) and all(torch.equal(a, b) for a, b in zip(got, want))
    twice = (keep.float() * 2).to(torch.bfloat16)
    got = ops.rmsnorm_mx8(keep, None, 1e-6, residual=keep)
    assert torch.equal(keep, twice) and all(torch.equal(a, b) for a, b in zip(got, ops.rmsnorm_mx8(twice, None, 1e-6)))
