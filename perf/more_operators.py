"""Measured cases of the operators on a KV cache held in 4 bits.

* ``store``: per-head RMS norms of q and k, rotation, and the store of k and v as 4-bit codes
  under one 8-bit scale per 32 dims, followed by the read-back of the stored rows;
* ``decode``: attention of one query token per request over the paged 4-bit cache;
* ``extend``: causal attention of several query tokens per request over the same cache, from a
  few (drafted) tokens to prompt chunks;
* ``copy``: copies of whole pages over every layer of a pool, for forks and for compaction.

The cache's numbers: a group of 32 consecutive dims of one token and head has a scale
s = (8 + m) 2^(e - 24), held as the byte 8 e + m, the smallest for which max |x| <= 7.5 s; an
element is s (c - 8) with a code c = clamp(round(x / s), -8, 7) + 8.

``run`` computes them in elementary torch operations while ``own`` is false and calls
``minisgl.ops`` when it is true.
"""

import math
import random

import torch

own = False

DEV = "cuda"
GROUP = 32  # dims under one scale


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of one request through a small model's layer (16 q heads, 8 kv heads): latency
        dict(name="store token", op="store", rows=1, hq=16, hk=8, d=128, page=64, norm=True),
        # a decode batch of a 32B dense model (64 / 8 heads)
        dict(name="store batch", op="store", rows=256, hq=64, hk=8, d=128, page=64, norm=True),
        # a prompt chunk, without norms, ragged number of rows
        dict(name="store chunk", op="store", rows=8189, hq=64, hk=8, d=128, page=64, norm=False),
        # one short request: latency
        dict(name="decode one short", op="decode", batch=1, longest=700, hq=16, hk=8, d=128, page=64),
        # one request of a long context: the split over the keys
        dict(name="decode one long", op="decode", batch=1, longest=131072, hq=64, hk=8, d=128, page=64),
        # a full running batch of ragged lengths
        dict(name="decode batch", op="decode", batch=256, longest=4096, hq=64, hk=8, d=128, page=64),
        # small pages, 64-dim heads, groups of 7 query heads
        dict(name="decode d64 ragged", op="decode", batch=33, longest=9001, hq=14, hk=2, d=64, page=16),
        # drafted tokens of a few requests, verified in one pass
        dict(name="extend drafted", op="extend", batch=8, q=5, longest=20011, hq=32, hk=8, d=128, page=64),
        # whole short prompts, ragged
        dict(name="extend prompts", op="extend", batch=6, q=1500, longest=1500, hq=32, hk=8, d=128, page=32),
        # a chunk of a long prompt behind what is cached already
        dict(name="extend chunk", op="extend", batch=1, q=2048, longest=16384, hq=64, hk=8, d=128, page=64),
        # forking one partly filled page of a small model's bf16 pool
        dict(name="copy fork", op="copy", pairs=1, layers=28, hk=8, d=128, page=64, bits=16),
        # compacting the 4-bit pool of a 64-layer model
        dict(name="copy compact", op="copy", pairs=500, layers=64, hk=8, d=128, page=64, bits=4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "extend", "extend", "copy"])
    hq, hk = rng.choice([(16, 8), (32, 8), (64, 8), (40, 8), (32, 4), (8, 1), (12, 12), (14, 2), (28, 4)])
    d = rng.choice([128, 128, 128, 64])
    page = rng.choice([16, 32, 64, 64, 128])
    heads = dict(hq=hq, hk=hk, d=d, page=page)
    if op == "store":
        return dict(op=op, rows=_log_int(rng, 1, min(16384, 8192 * 80 // (hq + 2 * hk))), norm=rng.random() < 0.5, **heads)
    if op == "decode":
        while True:
            batch, longest = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
            if batch * longest * hk * d <= 256 * 4096 * 8 * 128:
                return dict(op=op, batch=batch, longest=longest, **heads)
    if op == "extend":
        while True:
            batch, longest = _log_int(rng, 1, 16), _log_int(rng, 2, 65536)
            q = _log_int(rng, 1, min(longest, 4096))
            if batch * q * longest * hq <= 2048 * 16384 * 64 and batch * longest * hk <= 256 * 4096 * 8:
                return dict(op=op, batch=batch, q=q, longest=longest, **heads)
    layers, bits = rng.choice([1, 2, 28, 36, 48, 64]), rng.choice([4, 16])
    size = layers * hk * page * d * bits
    return dict(op=op, pairs=_log_int(rng, 1, max(1, 500 * 64 * 8 * 64 * 128 * 4 // size)), layers=layers, hk=hk, d=d,
                page=page, bits=bits)


def _lens(case):
    """Keys and query tokens of each request, a function of the case alone; the first is the longest."""
    rng = random.Random("%s %s %s" % (case["batch"], case["longest"], case.get("q", 1)))
    keys, queries = [case["longest"]], [case.get("q", 1)]
    for _ in range(case["batch"] - 1):
        keys.append(rng.randint(1, case["longest"]))
        queries.append(min(keys[-1], rng.randint(max(1, queries[0] // 2), queries[0])))
    return keys, queries


# ------------------------------------------------------------------ inputs
def _cache(g, pages, hk, page, d):
    """A filled cache in plain order: codes two per byte [2, pages, hk, page, d / 2] (even dim in
    the low nibble) and scale bytes [2, pages, hk, page, d / 32]; about unit variance."""
    packed = torch.empty(2, pages, hk, page, d // 2, dtype=torch.uint8, device=DEV)
    for kv in range(2):
        for lo in range(0, pages, 1024):
            n = min(1024, pages - lo)
            c = torch.randn(n, hk, page, d, generator=g, device=DEV, dtype=torch.float16)
            c = c.mul_(2.7).round_().clamp_(-8, 7).add_(8.0).to(torch.uint8)
            packed[kv, lo:lo + n] = c[..., 0::2] | (c[..., 1::2] << 4)
    sf = torch.randint(18 * 8 + 4, 20 * 8 + 2, (2, pages, hk, page, d // GROUP), generator=g, device=DEV)
    return packed, sf.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "copy":
        pages = 2 * case["pairs"] + 3
        order = torch.randperm(pages, generator=g, device=DEV).tolist()
        s["src"], s["dst"] = order[:case["pairs"]], order[case["pairs"]:2 * case["pairs"]]
        block = (case["hk"], case["page"], case["d"])
        if case["bits"] == 4:
            block = (case["hk"], case["page"] * (case["d"] // 2 + case["d"] // GROUP))
        shape = (2, case["layers"], pages) + block
        if case["bits"] == 4:
            s["pool"] = torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8)
        else:
            s["pool"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
        return s
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    if case["op"] == "store":
        rows = case["rows"]
        x = torch.randn(rows, (hq + 2 * hk) * d, generator=g, device=DEV)
        hot = torch.randint(0, x.shape[1], (x.shape[1] // 128,), generator=g, device=DEV)
        x[:, hot] *= 8.0  # a few channels of keys and values are far larger than the others
        s["qkv"] = x.to(torch.bfloat16)
        s["q_out"] = torch.empty(rows, hq * d, dtype=torch.bfloat16, device=DEV)
        pos = torch.randint(0, 32768, (rows,), generator=g, device=DEV)
        if rows > 256:  # a chunk: consecutive positions
            pos = pos[0] + torch.arange(rows, device=DEV)
        s["positions"] = pos.to(torch.int32)
        angle = torch.arange(49152, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2).double() / d)
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float().to(DEV)
        for name in ("q_norm", "k_norm"):
            w = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
            s[name] = w.to(torch.bfloat16) if case["norm"] else None
        pages = -(-rows // page) + 2
        at = torch.arange(rows, device=DEV)  # a chunk fills its pages in order, a decode batch has a page each
        pages = rows + 2 if rows <= 256 else pages
        order = torch.randperm(pages, generator=g, device=DEV)
        s["slots"] = (order[at] * page + pos % page if rows <= 256 else order[at // page] * page + at % page).to(torch.int32)
        if own:
            from minisgl.quant import kv4_block_bytes

            s["pool"] = torch.zeros(2, 1, pages, hk, kv4_block_bytes(page, d), dtype=torch.uint8, device=DEV)
        return s
    keys, queries = _lens(case)
    batch = len(keys)
    need = [-(-n // page) for n in keys]
    pages = sum(need) + 3
    packed, sf = _cache(g, pages, hk, page, d)
    order = torch.randperm(pages, generator=g, device=DEV)
    width = (max(keys) + 2 * page + 63) // 64 * 64
    table = torch.zeros(batch + 1, width, dtype=torch.int32, device=DEV)
    rows = torch.randperm(batch + 1, generator=g, device=DEV)[:batch]
    first = 0
    for row, n, p in zip(rows.tolist(), keys, need):
        at = torch.arange(n, device=DEV)
        table[row, :n] = (order[first + at // page] * page + at % page).to(torch.int32)
        first += p
    s["table"], s["req_rows"] = table, rows.to(torch.int32)
    s["seq_lens"] = torch.tensor(keys, dtype=torch.int32, device=DEV)
    total = sum(queries)
    # the q heads at the start of fused qkv rows
    s["qkv"] = (torch.randn(total, (hq + 2 * hk) * d, generator=g, device=DEV) * 1.3).to(torch.bfloat16)
    s["scale"] = d ** -0.5
    cu = [0]
    for n in queries:
        cu.append(cu[-1] + n)
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["max_q"] = max(queries)
    # where each query token's row lies in the padded batch of the plain form, and its position
    s["row_of"] = torch.cat([b * max(queries) + torch.arange(n) for b, n in enumerate(queries)]).to(DEV)
    if own:
        from minisgl import ops
        from minisgl.quant import pack_kv4

        s["pool"] = pack_kv4(packed, sf)[:, None].contiguous()
        if case["op"] == "extend":  # made once per batch, for every layer
            s["plan"] = ops.KV4PrefillPlan(keys, torch.device(DEV))
    else:
        s["packed"], s["sf"] = packed, sf
    return s


# ------------------------------------------------------------------ plain forms
def _plain_quantize(x):
    """Values of the codes of x [..., d] (fp32), as bf16 (which holds them exactly)."""
    b = x.unflatten(-1, (-1, GROUP))
    # a tensor as divisor: a number's reciprocal would be multiplied by, which misses where max |x| = 7.5 s
    need = b.abs().amax(-1, keepdim=True) / torch.full((1,), 7.5, device=x.device)
    mant, ex = torch.frexp(need)  # need = mant 2^ex; 16 mant in [8, 16), rounded up to whole steps
    step = torch.ldexp(torch.ceil(mant * 16.0), ex - 4).clamp(2.0 ** -21, 1920.0)
    return ((b / step).round().clamp(-8.0, 7.0) * step).flatten(-2).to(torch.bfloat16)


def _plain_rotate(x, w, cs, eps):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()
    a, b = x.chunk(2, dim=-1)
    c, s = cs.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_store(s):
    rows, hq, hk, d = s["rows"], s["hq"], s["hk"], s["d"]
    x = s["qkv"].float().view(rows, hq + 2 * hk, d)
    cs = s["cos_sin"][s["positions"].long()][:, None]
    q = _plain_rotate(x[:, :hq], s["q_norm"], cs, 1e-6)
    k = _plain_rotate(x[:, hq:hq + hk], s["k_norm"], cs, 1e-6)
    s["q_out"].copy_(q.reshape(rows, hq * d))
    return [s["q_out"], _plain_quantize(k), _plain_quantize(x[:, hq + hk:])]


def _plain_rows(s, kv, slots):
    """Rows [batch, keys, hk, d] of K or V in fp32."""
    hk, d, page = s["hk"], s["d"], s["page"]
    at, off = slots // page, slots % page
    c = s["packed"][kv][at, :, off]
    sf = s["sf"][kv][at, :, off].int()
    step = torch.ldexp((8 + sf % 8).float(), sf // 8 - 24)
    v = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).float() - 8.0
    return (v.unflatten(-1, (-1, GROUP)) * step[..., None]).flatten(-2)


def _plain_attention(s):
    hq, hk, d, batch, mq = s["hq"], s["hk"], s["d"], s["batch"], s["max_q"]
    slots = s["table"][s["req_rows"].long(), :s["longest"]].long()
    at = torch.arange(s["longest"], device=DEV)
    q = torch.zeros(batch * mq, hq * d, device=DEV)
    q[s["row_of"]] = s["qkv"][:, :hq * d].float()
    q = q.view(batch, mq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    score = (q @ _plain_rows(s, 0, slots).permute(0, 2, 3, 1)) * s["scale"]
    count = s["cu_q"].diff()
    last = (s["seq_lens"] - count)[:, None] + torch.arange(mq, device=DEV)  # position of each query token
    seen = at <= last[..., None]  # [batch, mq, keys]
    score = score.view(batch, hk, hq // hk, mq, -1).masked_fill_(~seen[:, None, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1)
    o = score.flatten(2, 3) @ _plain_rows(s, 1, slots).transpose(1, 2)
    o = o.view(batch, hk, hq // hk, mq, d) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * mq, hq * d)[s["row_of"]]
    return o.to(torch.bfloat16)


def _plain_copy(s):
    src, dst = (torch.tensor(v, device=DEV) for v in (s["src"], s["dst"]))
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    return s["pool"]


def run(state):
    s = state
    if own:
        from minisgl import ops

        if s["op"] == "copy":
            return ops.copy_pages(s["pool"], s["src"], s["dst"])
        hq, hk, d, page = s["hq"], s["hk"], s["d"], s["page"]
        if s["op"] == "store":
            ops.rope_store_kv4(s["qkv"], s["positions"], s["cos_sin"], s["q_norm"], s["k_norm"], s["pool"], 0,
                               s["slots"], hq, hk, d, page, 1e-6, q_out=s["q_out"])
            k, v = ops.load_kv4(s["pool"], 0, s["slots"], hk, d, page)
            return [s["q_out"], k, v]
        if s["op"] == "decode":
            return ops.decode_attention_kv4(s["qkv"], s["pool"], 0, s["table"], s["req_rows"], s["seq_lens"], hq, hk, d,
                                            page, s["scale"])
        return ops.prefill_attention_kv4(s["qkv"], s["pool"], 0, s["table"], s["req_rows"], s["seq_lens"], s["cu_q"],
                                         s["max_q"], hq, hk, d, page, s["scale"], plan=s["plan"])
    if s["op"] == "copy":
        return _plain_copy(s)
    return _plain_store(s) if s["op"] == "store" else _plain_attention(s)


# ------------------------------------------------------------------ work and exact values
def work(case):
    d = case["d"]
    held = case["hk"] * 2 * (d // 2 + d // GROUP)  # bytes of one token in the cache
    if case["op"] == "copy":
        row = held if case["bits"] == 4 else case["hk"] * 2 * d * 2
        return {"bytes": 2 * case["pairs"] * case["layers"] * case["page"] * row, "flops": 0}
    hq, hk = case["hq"], case["hk"]
    if case["op"] == "store":
        row = (hq + 2 * hk) * d * 2 + d * 4 + hq * d * 2 + 2 * held + 2 * hk * d * 2
        return {"bytes": case["rows"] * row, "flops": case["rows"] * (hq + 2 * hk) * d * 10}
    keys, queries = _lens(case)
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for k, n in zip(keys, queries))
    return {"bytes": sum(keys) * held + sum(queries) * hq * d * 4, "flops": 4 * pairs * hq * d}


def _exact_quantize(x):
    b = x.reshape(x.shape[:-1] + (-1, GROUP))
    top = b.abs().max(dim=-1).values
    table = torch.tensor([(8 + m) * 2.0 ** (e - 24) for e in range(32) for m in range(8)], dtype=torch.float64, device=DEV)
    step = table[torch.searchsorted(7.5 * table, top).clamp(max=255)][..., None]  # the smallest that reaches the largest
    return (torch.clamp(torch.round(b / step), -8, 7) * step).reshape(x.shape)


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    if case["op"] == "copy":
        return None
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    half = d // 2
    if case["op"] == "store":
        x = s["qkv"].double().reshape(case["rows"], hq + 2 * hk, d)
        cs = s["cos_sin"].double()[s["positions"].long()][:, None, :]
        turned = []
        for part, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hk], s["k_norm"])):
            if w is not None:
                part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            z = torch.complex(part[..., :half], part[..., half:]) * torch.complex(cs[..., :half], cs[..., half:])
            turned.append(torch.cat([z.real, z.imag], dim=-1))
        return [turned[0].reshape(case["rows"], hq * d), _exact_quantize(turned[1]), _exact_quantize(x[:, hq + hk:])]
    keys, queries = _lens(case)
    out, first = [], 0
    for b, (n, m) in enumerate(zip(keys, queries)):
        slot = s["table"][int(s["req_rows"][b]), :n].long()
        kv = []
        for part in range(2):
            c = s["packed"][part][slot // page, :, slot % page].int()
            f = s["sf"][part][slot // page, :, slot % page].double()
            e = torch.floor(f / 8)
            v = torch.empty(n, hk, d, dtype=torch.float64, device=DEV)
            v[..., 0::2], v[..., 1::2] = (c % 16).double() - 8, (c // 16).double() - 8
            v = v * ((8 + f - 8 * e) * torch.exp2(e - 24)).repeat_interleave(GROUP, dim=-1)
            kv.append(v)
        q = s["qkv"][first:first + m, :hq * d].double().reshape(m, hk, hq // hk, d)
        rows = torch.empty(m, hk, hq // hk, d, dtype=torch.float64, device=DEV)
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None]
        for h in range(hk):
            sc = torch.einsum("mgd,nd->gmn", q[:, h], kv[0][:, h]) * s["scale"]
            p = torch.softmax(sc.masked_fill(hidden, -math.inf), dim=-1)
            rows[:, h] = torch.einsum("gmn,nd->mgd", p, kv[1][:, h])
        out.append(rows.reshape(m, hq * d))
        first += m
    return torch.cat(out)
