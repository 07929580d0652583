"""Measured cases of the operators on quantised operands.

* ``int4_linear``: products with 4-bit weights under group scales (and zero points), from one
  token to a prompt chunk, for bf16, fp16 and MXFP8 rows;
* ``rmsnorm_mx8``: residual addition + RMSNorm whose output is MXFP8 (E4M3 elements, one
  power-of-two E8M0 scale per 32);
* ``act_mx8``: silu(gate) * up or gelu(gate) * up with the same output.

``run`` computes them in elementary torch operations while ``own`` is false and calls
``minisgl.ops`` when it is true.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32  # elements under one E8M0 scale
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    lin = dict(op="int4_linear", zeros=False, bias=False)
    return [
        # one token through a small model's projection: latency
        dict(lin, name="linear token small", rows=1, n=2048, k=1024, group=128, x="bf16"),
        # one token through the gate|up projection of a 32B dense model (5120 -> 2 x 25600): the weight stream
        dict(lin, name="linear token gate_up", rows=1, n=51200, k=5120, group=128, x="bf16"),
        # a decode batch through its down projection, zero points as asymmetric checkpoints have them
        dict(lin, name="linear batch down fp16", rows=8, n=5120, k=25600, group=128, zeros=True, x="fp16"),
        # odd sizes: a vocabulary-like ragged N, K that ends inside a group, small groups, a bias
        dict(lin, name="linear ragged", rows=3, n=12301, k=4168, group=32, zeros=True, bias=True, x="bf16"),
        # MXFP8 rows (what rmsnorm_mx8 writes) of a larger decode batch
        dict(lin, name="linear batch mx8", rows=24, n=7168, k=8192, group=64, x="mx8"),
        # a prompt chunk: bound by the tensor cores
        dict(lin, name="linear prompt", rows=2000, n=8192, k=7168, group=128, x="bf16"),
        # one token's row: latency
        dict(name="norm token", op="rmsnorm_mx8", rows=1, cols=5120, type="bf16", residual=True),
        # a prompt chunk of a wide model: memory
        dict(name="norm prompt", op="rmsnorm_mx8", rows=8192, cols=7168, type="bf16", residual=True),
        # the first norm of a stack (no residual yet), an odd number of rows and of 32-blocks
        dict(name="norm first fp16", op="rmsnorm_mx8", rows=777, cols=4128, type="fp16", residual=False),
        # a decode batch's activation
        dict(name="act batch", op="act_mx8", act="silu", rows=64, cols=25600, type="bf16", interleaved=False),
        # a prompt chunk's activation, gate|up in alternating blocks of 64 as the model layers keep them
        dict(name="act prompt", op="act_mx8", act="silu", rows=4096, cols=25600, type="bf16", interleaved=True),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["int4_linear", "int4_linear", "rmsnorm_mx8", "act_mx8"])
    if op == "int4_linear":
        x = rng.choice(["bf16", "bf16", "fp16", "mx8"])
        while True:
            rows = _log_int(rng, 1, 2000) if rng.random() < 0.4 else rng.randint(1, 32)
            n = _log_int(rng, 256, 51200)
            k = _log_int(rng, 256, 25600, 32 if x == "mx8" else 8)
            if n * k <= 51200 * 5120 and rows * n * k <= 2000 * 8192 * 7168:
                break
        return dict(op=op, rows=rows, n=n, k=k, group=rng.choice([32, 64, 128, 128]), zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.25, x=x)
    cols = _log_int(rng, 512, 16384, 32)
    if op == "rmsnorm_mx8":
        rows = min(_log_int(rng, 1, 16384), 8192 * 7168 // cols)
        return dict(op=op, rows=rows, cols=cols, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    residual=rng.random() < 0.7)
    act = rng.choice(["silu", "silu", "gelu"])
    interleaved = act == "silu" and rng.random() < 0.5
    if interleaved:
        cols = cols // 64 * 64
    rows = min(_log_int(rng, 1, 8192), 4096 * 25600 // cols)
    return dict(op=op, act=act, rows=rows, cols=cols, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                interleaved=interleaved)


# ------------------------------------------------------------------ inputs
def _rows_with_outliers(g, rows, cols, scale):
    """Activations: normal, with a few channels that are 20 times larger, as residual streams have them."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * scale
    hot = torch.randint(0, cols, (max(1, cols // 512),), generator=g, device=DEV)
    x[:, hot] *= 20.0
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "int4_linear":
        rows, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        groups = -(-k // group)
        # codes of round-to-nearest quantisation of normal weights: about normal around the middle
        codes = torch.randn(n, k, generator=g, device=DEV, dtype=torch.float16).mul_(2.7).add_(8.0).round_()
        codes = codes.clamp_(0, 15).to(torch.uint8)
        packed = codes[:, 0::2] | (codes[:, 1::2] << 4)  # element 2i in the low nibble of byte i
        del codes
        st = torch.float16 if case["x"] == "fp16" else torch.bfloat16
        scales = (torch.rand(n, groups, generator=g, device=DEV) * 0.008 + 0.002).to(st)
        zeros = torch.randint(5, 12, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        x = _rows_with_outliers(g, rows, k, 1.0)
        s["x_scales"] = None
        if case["x"] == "mx8":
            b = x.view(rows, k // BLOCK, BLOCK)
            e = torch.ceil(torch.log2(b.abs().amax(-1) / 448.0))
            s["x_rows"] = torch.ldexp(b, -e[..., None]).view(rows, k).to(torch.float8_e4m3fn).view(torch.uint8)
            s["x_scales"] = (e + 127).to(torch.uint8)
        else:
            s["x_rows"] = x.to(st)
        s["bias_row"] = torch.randn(n, generator=g, device=DEV).to(st) if case["bias"] else None
        if own:  # the layout that a program makes once, when it loads its weights
            from minisgl.quant import int4_weight

            s["weight"] = int4_weight(packed, scales, zeros, group)
        else:
            s["packed"], s["scales"], s["zero_points"] = packed, scales, zeros
        return s
    dt = TYPES[case["type"]]
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "rmsnorm_mx8":
        s["x_rows"] = _rows_with_outliers(g, rows, cols, 1.0).to(dt)
        s["weight"] = (1.0 + 0.1 * torch.randn(cols, generator=g, device=DEV)).to(dt)
        s["stream"] = _rows_with_outliers(g, rows, cols, 3.0).to(dt) if case["residual"] else None
        s["stream_out"] = torch.empty_like(s["stream"]) if case["residual"] else None
        if rows > 8:  # padding rows of a batch are zero
            s["x_rows"][-1] = 0
            if case["residual"]:
                s["stream"][-1] = 0
    else:
        s["x_rows"] = (torch.randn(rows, 2 * cols, generator=g, device=DEV) * 1.5).to(dt)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_int4_linear(s):
    packed, group = s["packed"], s["group"]
    n, k = s["n"], s["k"]
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).view(n, k).float()
    pad = -k % group
    if pad:
        codes = torch.cat([codes, codes.new_zeros(n, pad)], dim=1)
    codes = codes.view(n, -1, group)
    codes = codes - (s["zero_points"].float()[..., None] if s["zero_points"] is not None else 8.0)
    w = (codes * s["scales"].float()[..., None]).view(n, k + pad)[:, :k]
    x = s["x_rows"]
    if s["x_scales"] is not None:
        x = x.view(torch.float8_e4m3fn).float().view(s["rows"], k // BLOCK, BLOCK)
        x = torch.ldexp(x, s["x_scales"].float()[..., None] - 127.0).view(s["rows"], k)
    y = x.float() @ w.t()
    if s["bias_row"] is not None:
        y = y + s["bias_row"].float()
    return y.to(s["scales"].dtype)


def _plain_mx8(y):
    rows, cols = y.shape
    b = y.view(rows, cols // BLOCK, BLOCK)
    amax = b.abs().amax(-1)
    mant, ex = torch.frexp(amax)  # amax = mant 2^ex, mant in [0.5, 1); 448 = 0.875 * 2^9
    e = ex - 9 + (mant > 0.875)
    byte = torch.where(amax > 0, (e + 127).clamp(1, 254), 0)
    q = torch.ldexp(b, (127 - byte)[..., None]).view(rows, cols)
    return q.to(torch.float8_e4m3fn), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_rmsnorm_mx8(s):
    v = s["x_rows"].float()
    if s["stream"] is not None:
        v = (v + s["stream"].float()).to(s["x_rows"].dtype)
        s["stream_out"].copy_(v)
        v = v.float()
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    q, sf = _plain_mx8(y)
    return [q, sf] if s["stream"] is None else [q, sf, s["stream_out"]]


def _plain_act_mx8(s):
    x = s["x_rows"].float()
    rows, cols = s["rows"], s["cols"]
    if s["interleaved"]:
        x = x.view(rows, cols // 64, 2, 64).transpose(1, 2)
    x = x.reshape(rows, 2, cols)
    gate, up = x[:, 0], x[:, 1]
    if s["act"] == "silu":
        y = gate / (1.0 + torch.exp(-gate)) * up
    else:
        y = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5))) * up
    return list(_plain_mx8(y))


def _mx8_values(q, sf):
    """The outputs as the numbers that their bits stand for: E4M3 elements and power-of-two scales."""
    return [q.view(torch.float8_e4m3fn), sf.view(torch.float8_e8m0fnu)]


def run(state):
    s = state
    if own:
        from minisgl import ops

        if s["op"] == "int4_linear":
            return ops.int4_linear(s["x_rows"], s["weight"], s["bias_row"], x_scales=s["x_scales"])
        if s["op"] == "rmsnorm_mx8":
            q, sf = ops.rmsnorm_mx8(s["x_rows"], s["weight"], 1e-6, residual=s["stream"],
                                    residual_out=s["stream_out"])
            return _mx8_values(q, sf) + ([] if s["stream"] is None else [s["stream_out"]])
        if s["act"] == "silu":
            return _mx8_values(*ops.silu_and_mul_mx8(s["x_rows"], interleaved=s["interleaved"]))
        return _mx8_values(*ops.gelu_and_mul_mx8(s["x_rows"]))
    if s["op"] == "int4_linear":
        return _plain_int4_linear(s)
    return _plain_rmsnorm_mx8(s) if s["op"] == "rmsnorm_mx8" else _plain_act_mx8(s)


# ------------------------------------------------------------------ work and exact values
def work(case):
    if case["op"] == "int4_linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        groups = -(-k // case["group"])
        weight = n * k / 2 + n * groups * (2.5 if case["zeros"] else 2)
        x = rows * k * (1 + 1 / BLOCK if case["x"] == "mx8" else 2)
        return {"bytes": weight + x + rows * n * 2 + (2 * n if case["bias"] else 0), "flops": 2 * rows * n * k}
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["type"] == "fp32" else 2
    q = rows * cols * (1 + 1 / BLOCK)
    if case["op"] == "rmsnorm_mx8":
        return {"bytes": rows * cols * size * (3 if case["residual"] else 1) + cols * size + q,
                "flops": rows * cols * 8}
    return {"bytes": rows * cols * 2 * size + q, "flops": rows * cols * 12}


def _exact_mx8(y):
    rows, cols = y.shape
    b = y.reshape(rows, -1, BLOCK)
    ratio = b.abs().amax(-1) / 448.0
    m, ex = torch.frexp(ratio)
    e = (ex - (m == 0.5).to(ex.dtype)).double().clamp(-126, 127)  # smallest e with ratio <= 2^e
    e = torch.where(ratio > 0, e, torch.full_like(e, -127.0))
    v = torch.where((ratio > 0)[..., None], b * torch.exp2(-e)[..., None], torch.zeros_like(b))
    step = torch.exp2(torch.frexp(v)[1].double().sub(1).clamp(min=-6) - 3)  # 3 mantissa bits, subnormals below 2^-6
    v = torch.round(v / step) * step  # half to even
    return [v.reshape(rows, cols), torch.exp2(e)]


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    if case["op"] == "int4_linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        x = s["x_rows"]
        if s["x_scales"] is not None:
            x = x.view(torch.float8_e4m3fn).double()
            x = x * torch.exp2(s["x_scales"].double() - 127).repeat_interleave(BLOCK, dim=1)
        x = x.double()
        y = torch.empty(rows, n, dtype=torch.float64, device=DEV)
        group_of = torch.arange(k, device=DEV) // case["group"]
        for lo in range(0, n, 8192):
            p = s["packed"][lo:lo + 8192].to(torch.int32)
            w = torch.empty(p.shape[0], k, dtype=torch.float64, device=DEV)
            w[:, 0::2] = (p % 16).double()
            w[:, 1::2] = (p // 16).double()
            z = s["zero_points"][lo:lo + 8192].double()[:, group_of] if case["zeros"] else 8.0
            w = (w - z) * s["scales"][lo:lo + 8192].double()[:, group_of]
            y[:, lo:lo + 8192] = x @ w.t()
        return y + s["bias_row"].double() if case["bias"] else y
    x = s["x_rows"]
    if case["op"] == "rmsnorm_mx8":
        out = []
        v = x.double()
        if case["residual"]:
            total = x.double() + s["stream"].double()
            v = total.to(x.dtype).double()  # the residual stream is kept in the activation's type
            out = [total]
        y = v / torch.sqrt((v * v).sum(-1, keepdim=True) / case["cols"] + 1e-6) * s["weight"].double()
        return _exact_mx8(y) + out
    rows, cols = case["rows"], case["cols"]
    x = x.double()
    if case["interleaved"]:
        at = torch.arange(cols, device=DEV)
        at = at // 64 * 128 + at % 64
        gate, up = x[:, at], x[:, at + 64]
    else:
        gate, up = x[:, :cols], x[:, cols:]
    act = gate * torch.sigmoid(gate) if case["act"] == "silu" else gate * torch.special.ndtr(gate)
    return _exact_mx8(act * up)
