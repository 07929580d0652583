"""Plain float64 statements of the operators on the 4-bit KV cache, written from the format's
formulas, and the bounds that their kernels are held to."""

import math

import torch

from minisgl.quant import pack_kv4


def scales(sf):
    sf = sf.double()
    e = torch.floor(sf / 8)
    return (8 + sf - 8 * e) * torch.exp2(e - 24)


def values(packed, sf):
    """Plain-order codes [..., d / 2] and scale bytes [..., d / 32] -> float64 [..., d]."""
    p = packed.to(torch.int32)
    c = torch.stack([p % 16, p // 16], dim=-1).flatten(-2).double() - 8
    return c * scales(sf).repeat_interleave(32, dim=-1)


def quantize(x):
    """Rows [..., d] -> (codes 0..15, scale bytes) by search over the format's scales."""
    b = x.double().reshape(x.shape[:-1] + (-1, 32))
    table = scales(torch.arange(256))
    top = b.abs().amax(-1)
    byte = (7.5 * table < top[..., None]).sum(-1).clamp(max=255)  # the first that reaches the largest
    c = torch.round(b / table[byte][..., None]).clamp(-8, 7) + 8
    return c.reshape(x.shape).to(torch.uint8), byte.to(torch.uint8)


def make_cache(lens, hk, d, page, layers=2, seed=0, sf_range=(148, 162), extra_rows=2, spare=3):
    """(packed, sf, pool, page_table, req_rows) on the CPU: random codes in every slot of every
    page, table rows in shuffled order, what lies past a request's end pointing at other pages."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + spare
    packed = torch.randint(0, 256, (2, layers, pages, hk, page, d // 2), generator=g, dtype=torch.uint8)
    sf = torch.randint(*sf_range, (2, layers, pages, hk, page, d // 32), generator=g).to(torch.uint8)
    width = max(64, (max(lens) + page + 63) // 64 * 64)
    table = torch.randint(0, pages * page, (len(lens) + extra_rows, width), generator=g).to(torch.int32)
    order = torch.randperm(pages, generator=g)
    rows = torch.randperm(len(lens) + extra_rows, generator=g)[:len(lens)].to(torch.int32)
    first = 0
    for row, n, k in zip(rows.tolist(), lens, need):
        at = torch.arange(n)
        table[row, :n] = (order[first + at // page] * page + at % page).to(torch.int32)
        first += k
    return packed, sf, pack_kv4(packed, sf), table, rows


def attention(q, packed, sf, layer, table, rows, lens, queries, hq, hk, scale):
    """(out, bound) float64 [T, hq, d] of causal attention; q [T, hq, d] as float64.

    Bound: the output's rounding to bf16 (2^-8 |out|), that of every weight p to bf16 (2^-8 of
    sum p |v|), and the error of the scores, which weights take on twice (numerator and sum).
    Few rows: a group's 32 products q c are two tensor-core sums of 16 + 1 terms no larger than
    15 sum |q|, each kept to 2^-23, the offset of all groups, -8 s sum(q), one such sum, and
    five more sums are kept to 2^-24: (2 * 17 * 15 + 17 * 8 + 5 * 23 / 2) 2^-23 s sum |q| = 704.
    Many rows: 128 products q s (c - 8) in eight tensor-core sums, 8 * 17 * 8 = 1088. So 1100."""
    page = packed.shape[-2]
    k_all, v_all = values(packed[0, layer], sf[0, layer]), values(packed[1, layer], sf[1, layer])
    s_all = scales(sf[0, layer])
    G = hq // hk
    out, bound, first = [], [], 0
    for row, n, m in zip(rows.tolist(), lens, queries):
        at = table[row, :n].long()
        k, v, s = (x[at // page, :, at % page] for x in (k_all, v_all, s_all))  # [n, hk, .]
        qb = q[first:first + m].reshape(m, hk, G, q.shape[-1])
        first += m
        o = torch.zeros(m, hk, G, q.shape[-1], dtype=torch.float64)
        e = torch.zeros_like(o)
        for i in range(m):
            seen = n - m + i + 1
            if seen <= 0:
                continue
            sc = torch.einsum("hgd,lhd->hgl", qb[i], k[:seen]) * scale
            p = torch.softmax(sc, dim=-1)
            o[i] = torch.einsum("hgl,lhd->hgd", p, v[:seen])
            a = torch.einsum("hgl,lhd->hgd", p, v[:seen].abs())
            reach = torch.einsum("hgx,lhx->hgl", qb[i].abs().reshape(hk, G, -1, 32).sum(-1), s[:seen])
            es = (reach * 1100 * 2.0 ** -23 * scale).amax(-1, keepdim=True)
            e[i] = 2.0 ** -8 * o[i].abs() + (2.0 ** -8 + 2.0 ** -20 + 2 * es) * a
        out.append(o.reshape(m, hq, q.shape[-1]))
        bound.append(e.reshape(m, hq, q.shape[-1]))
    return torch.cat(out), torch.cat(bound)


def rope_rows(x, w, cs, eps=1e-6):
    """Norm and rotation of x [T, heads, d] in float64; cs [T, d]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h], x[..., h:]) * torch.complex(cs[:, None, :h].double(), cs[:, None, h:].double())
    return torch.cat([z.real, z.imag], dim=-1)


def cos_sin(n, d, base=1e6):
    a = torch.arange(n).double()[:, None] * base ** (-torch.arange(0, d, 2).double() / d)
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def log_lens(batch, longest, seed):
    g = torch.Generator().manual_seed(seed)
    return [longest] + [max(1, int(math.exp(float(torch.rand((), generator=g)) * math.log(longest))))
                        for _ in range(batch - 1)]
