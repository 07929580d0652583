"""Kernels of the 4-bit KV cache against float64 statements."""

import pytest
import torch

from minisgl import ops
from minisgl.quant import pack_kv4, unpack_kv4

import kv4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _done():
    torch.cuda.synchronize()
    ops.check_device_errors(torch.device(DEV))


def _check(got, want, bound):
    err = (got.double().cpu() - want).abs()
    worst = (err - bound).max().item()
    assert (err <= bound + 1e-30).all(), f"beyond the bound by {worst:.3g}; largest error {err.max().item():.3g}"


# ------------------------------------------------------------- rows in and out
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hk,T", [(1, 1), (2, 5), (8, 130), (3, 67)])
def test_store_and_load_are_exact(d, page, hk, T):
    g = torch.Generator().manual_seed(T)
    pages = 2 * T // page + 3
    kv = (torch.randn(2, T, hk * d, generator=g) * torch.exp2(torch.randint(-12, 9, (2, T, hk * d // 32, 1), generator=g))
          .expand(-1, -1, -1, 32).flatten(-2)).to(torch.bfloat16)
    start = torch.randint(0, 256, (2, 2, pages, hk, page * (d // 2 + d // 32)), generator=g, dtype=torch.uint8)
    pool = start.to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    ops.store_kv4(kv[0].to(DEV), kv[1].to(DEV), pool, 1, slots.to(DEV), hk, d, page)
    k, v = ops.load_kv4(pool, 1, slots.to(DEV), hk, d, page)
    _done()
    packed, sf = unpack_kv4(pool.cpu(), page, d)
    was_packed, was_sf = unpack_kv4(start, page, d)
    at = slots.long()
    for i, back in enumerate((k, v)):
        codes, byte = oracle.quantize(kv[i].view(T, hk, d))
        want = codes[..., 0::2] | (codes[..., 1::2] << 4)
        assert torch.equal(packed[i, 1][at // page, :, at % page], want)
        assert torch.equal(sf[i, 1][at // page, :, at % page], byte)
        assert torch.equal(back.double().cpu(), oracle.values(want, byte))
    # every other row, and the other layer, as they were
    packed[:, 1, at // page, :, at % page] = was_packed[:, 1, at // page, :, at % page]
    sf[:, 1, at // page, :, at % page] = was_sf[:, 1, at // page, :, at % page]
    assert torch.equal(packed, was_packed) and torch.equal(sf, was_sf)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("T", [3, 4, 9, 64])
def test_store_of_runs(offset, T):
    """Consecutive slots from any place of a group of four; two runs that meet inside a group."""
    d, hk, page = 128, 2, 16
    g = torch.Generator().manual_seed(T)
    x = torch.randn(2, T, hk * d, generator=g).to(torch.bfloat16)
    pool = torch.zeros(2, 1, 9, hk, page * 68, dtype=torch.uint8, device=DEV)
    slots = offset + torch.arange(T)
    slots[T // 2:] += 33
    ops.store_kv4(x[0].to(DEV), x[1].to(DEV), pool, 0, slots.to(torch.int32).to(DEV), hk, d, page)
    k, v = ops.load_kv4(pool, 0, slots.to(torch.int32).to(DEV), hk, d, page)
    _done()
    for want, got in zip(x, (k, v)):
        c, byte = oracle.quantize(want.view(T, hk, d))
        assert torch.equal(got.double().cpu(), oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte))


def test_store_of_special_values():
    d, hk, page = 64, 1, 16
    x = torch.zeros(6, d)
    x[0, 3] = float("inf")
    x[1, 5], x[1, 6] = float("-inf"), 3.0
    x[2, 7], x[2, 8] = float("nan"), 1.0
    x[3, :] = 1e30
    x[4, 0] = 1e-30
    x = x.to(torch.bfloat16)
    pool = torch.zeros(2, 1, 2, hk, page * 34, dtype=torch.uint8, device=DEV)
    slots = torch.arange(6, dtype=torch.int32, device=DEV)
    ops.store_kv4(x.to(DEV), x.to(DEV), pool, 0, slots, hk, d, page)
    k, v = ops.load_kv4(pool, 0, slots, hk, d, page)
    _done()
    assert torch.equal(k, v) and torch.isfinite(k).all()
    k = k[:, 0].float().cpu()
    assert k[0, 3] == 7 * 1920 and k[1, 5] == -8 * 1920 and k[1, 6] == 0
    assert k[2, 7] == 0 and abs(k[2, 8] - 1) < 1 / 13 and (k[3] == 7 * 1920).all()
    assert (k[4] == 0).all() and (k[5] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(16, 8), (7, 1), (4, 4)])
@pytest.mark.parametrize("T,norm", [(1, True), (37, False), (600, True)])
@pytest.mark.parametrize("in_place", [True, False])
def test_rope_store(d, hq, hk, T, norm, in_place):
    page = 32
    g = torch.Generator().manual_seed(T + d)
    qkv = torch.randn(T, (hq + 2 * hk) * d + 8, generator=g).to(torch.bfloat16)
    cs = oracle.cos_sin(4096, d)
    pos = torch.randint(0, 4096, (T,), generator=g).to(torch.int32)
    w = (1 + 0.2 * torch.randn(2, d, generator=g)).to(torch.bfloat16)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    pool = torch.zeros(2, 2, pages, hk, page * (d // 2 + d // 32), dtype=torch.uint8, device=DEV)
    x = qkv.to(DEV)
    q_out = None if in_place else torch.full((T, hq * d), 7.0, dtype=torch.bfloat16, device=DEV)
    weights = [v.to(DEV) if norm else None for v in w]
    ops.rope_store_kv4(x, pos.to(DEV), cs.to(DEV), *weights, pool, 1, slots.to(DEV), hq, hk, d, page, 1e-6, q_out=q_out)
    k, v = ops.load_kv4(pool, 1, slots.to(DEV), hk, d, page)
    _done()
    rows = qkv[:, :(hq + 2 * hk) * d].view(T, hq + 2 * hk, d)
    q_got = (x[:, :hq * d] if in_place else q_out).cpu().double().view(T, hq, d)
    if in_place:
        assert torch.equal(x[:, hq * d:].cpu(), qkv[:, hq * d:])
    else:
        assert torch.equal(x.cpu(), qkv)
    q = oracle.rope_rows(rows[:, :hq], w[0] if norm else None, cs[pos.long()])
    pair = q.abs() + q.abs().roll(d // 2, dims=-1)  # both terms of a rotation are below the pair's length
    _check(q_got, q, 2.0 ** -8 * q.abs() + 24 * 2.0 ** -24 * 2 * pair)
    kr = oracle.rope_rows(rows[:, hq:hq + hk], w[1] if norm else None, cs[pos.long()])
    kr32 = kr.abs().reshape(T, hk, -1, 32).amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(T, hk, d)
    # at most half a step from the row: a step is below 1.125 / 7.5 of the group's largest
    _check(k.double().cpu(), kr, kr32 * (1.125 / 15 + 2.0 ** -18))
    # and the codes those of the formula but where fp32 leaves a border's side open
    c, byte = oracle.quantize(kr)
    want = oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte)
    assert (k.double().cpu() != want).double().mean() < 1e-3
    c, byte = oracle.quantize(rows[:, hq + hk:])
    assert torch.equal(v.double().cpu(), oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte))


def test_bad_slots_and_positions_are_reported():
    d, hk, page = 128, 2, 16
    x = torch.randn(3, hk * d, device=DEV).to(torch.bfloat16)
    pool = torch.zeros(2, 1, 2, hk, page * 68, dtype=torch.uint8, device=DEV)
    slots = torch.tensor([5, -1, 32], dtype=torch.int32, device=DEV)
    ops.store_kv4(x, x, pool, 0, slots, hk, d, page)
    with pytest.raises(ops.DeviceIndexError):
        _done()
    k, _ = ops.load_kv4(pool, 0, slots, hk, d, page)
    with pytest.raises(ops.DeviceIndexError):
        _done()
    assert (k[0] != 0).any() and (k[1:] == 0).all()
    qkv = torch.randn(1, 4 * d, device=DEV).to(torch.bfloat16)
    ops.rope_store_kv4(qkv, torch.tensor([9], dtype=torch.int32, device=DEV), oracle.cos_sin(9, d).to(DEV), None, None,
                       pool[:, :, :, :1].contiguous(), 0, slots[:1], 2, 1, d, page, 1e-6)
    with pytest.raises(ops.DeviceIndexError):
        _done()


# ------------------------------------------------------------------ attention
def _attend(lens, queries, hq, hk, d, page, seed=0, q_scale=1.3, few=True, stride=8, **cache):
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page, seed=seed, **cache)
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(queries)
    q = (torch.randn(T, hq * d + stride, generator=g) * q_scale).to(torch.bfloat16)
    seq = torch.tensor(lens, dtype=torch.int32)
    cu = torch.tensor([0] + list(torch.tensor(queries).cumsum(0)), dtype=torch.int32)
    scale = d ** -0.5
    if all(n == 1 for n in queries) and few is not None:
        got = ops.decode_attention_kv4(q.to(DEV), pool.to(DEV), 1, table.to(DEV), rows.to(DEV), seq.to(DEV), hq, hk, d,
                                       page, scale)
    else:
        got = ops.prefill_attention_kv4(q.to(DEV), pool.to(DEV), 1, table.to(DEV), rows.to(DEV), seq.to(DEV), cu.to(DEV),
                                        max(queries), hq, hk, d, page, scale)
    _done()
    want, bound = oracle.attention(q[:, :hq * d].double().view(T, hq, d), packed, sf, 1, table, rows, lens, queries, hq,
                                   hk, scale)
    return got.view(T, hq, d), want, bound


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(16, 8), (64, 8), (4, 4), (7, 1), (40, 4), (16, 1)])
def test_decode(d, page, hq, hk):
    lens = [1, 2, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]
    _check(*_attend(lens, [1] * len(lens), hq, hk, d, page))


@pytest.mark.parametrize("lens", [[1], [128], [5000], [20000, 1], [3] * 300, [700] * 40], ids=lambda x: f"{len(x)}x{x[0]}")
def test_decode_splits(lens):
    """One request over many CTAs, many requests in one CTA."""
    _check(*_attend(lens, [1] * len(lens), 8, 1, 128, 64))


def test_decode_without_keys():
    got, want, bound = _attend([0, 5, 0], [1, 1, 1], 8, 2, 128, 16)
    _check(got, want, bound)
    assert (got[0] == 0).all() and (got[2] == 0).all()


@pytest.mark.parametrize("q_scale", [1e-3, 20.0])
def test_decode_flat_and_peaked(q_scale):
    _check(*_attend([900, 77], [1, 1], 8, 1, 128, 64, q_scale=q_scale))


def test_decode_scores_that_rise():
    """The running maximum moves with every tile: keys grow along the sequence."""
    lens, d, page = [2000], 128, 16
    packed, sf, pool, table, rows = oracle.make_cache(lens, 1, d, page, layers=1, sf_range=(120, 121))
    at = table[rows.long()[0], :2000].long()
    sf[0, 0, at // page, :, at % page] = (100 + 60 * torch.arange(2000) // 2000).to(torch.uint8)[:, None, None]
    q = (torch.randn(1, 8 * d, generator=torch.Generator().manual_seed(5)) * 30).to(torch.bfloat16)
    got = ops.decode_attention_kv4(q.to(DEV), pack_kv4(packed, sf).to(DEV), 0, table.to(DEV), rows.to(DEV),
                                   torch.tensor(lens, dtype=torch.int32, device=DEV), 8, 1, d, page, d ** -0.5)
    _done()
    want, bound = oracle.attention(q.double().view(1, 8, d), packed, sf, 0, table, rows, lens, [1], 8, 1, d ** -0.5)
    _check(got.view(1, 8, d), want, bound)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (128, 16), (64, 256)])
@pytest.mark.parametrize("hq,hk", [(8, 8), (32, 8), (7, 1), (32, 1)])
def test_extend_few_rows(d, page, hq, hk):
    lens, queries = [5, 70, 500, 129, 4, 9], [5, 3, 4, 1, 4, 2]
    if hq // hk * 5 > ops.KV4_FEW_ROWS:
        lens, queries = lens[1:], [2, 2, 1, 2, 2]
    _check(*_attend(lens, queries, hq, hk, d, page, few=None))


def test_extend_with_more_queries_than_keys():
    got, want, bound = _attend([3, 0, 200], [5, 2, 3], 8, 2, 128, 16, few=None)
    _check(got, want, bound)
    assert (got[:2] == 0).all() and (got[5:7] == 0).all()


@pytest.mark.parametrize("d,page", [(128, 16), (128, 64), (128, 256), (64, 32), (64, 128)])
@pytest.mark.parametrize("hq,hk", [(8, 8), (16, 2), (14, 2)])
def test_extend_many_rows(d, page, hq, hk):
    """The expanded path. A quarter of its weights come from a polynomial that is off by 7.5e-5,
    twice (numerator and sum), and its products keep n keys' sums to (17 / 16) n 2^-23, 1.6e-4 for
    1300 keys: together 0.08 of the 2^-8 of the weights' rounding."""
    lens, queries = [700, 150, 260], [300, 150, 1]
    got, want, bound = _attend(lens, queries, hq, hk, d, page, few=None)
    _check(got, want, 1.1 * bound)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [1, 3, 100], ids=["one token", "few rows", "many rows"])
def test_as_many_requests_as_a_call_takes(d, first):
    lens = [130] + [1 + i % 20 for i in range(ops.KV4_MAX_BATCH - 1)]
    got, want, bound = _attend(lens, [first] + [1] * (len(lens) - 1), 2, 2, d, 16)
    _check(got, want, 1.1 * bound)
    x = torch.zeros(len(lens) + 1, dtype=torch.int32, device=DEV)
    pool = torch.zeros(2, 1, 1, 2, 16 * (d // 2 + d // 32), dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match="at most"):
        ops.decode_attention_kv4(torch.zeros(len(lens) + 1, 2 * d, dtype=torch.bfloat16, device=DEV), pool, 0,
                                 x[:16].view(1, 16).contiguous(), x, x, 2, 2, d, 16, 0.1)


def test_extend_of_more_heads_than_a_tile_has_rows():
    _check(*_attend([40, 9], [3, 9], 130, 1, 64, 16, few=None))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("queries", [[3, 1], [150, 20]], ids=["few", "many"])
def test_extend_of_nothing(d, queries):
    """No request has a key: zeros, by either path (the plan of the second has no rows)."""
    got, _, _ = _attend([0, 0], queries, 4, 1, d, 16, few=None)
    assert (got == 0).all()


@pytest.mark.parametrize("queries", [[2, 1], [90, 40]], ids=["few", "many"])
def test_rows_behind_the_last_request(queries):
    """Padded rows of q are read by nobody's product and their rows of out stay as they are."""
    lens, hq, hk, d, page = [200, 130], 8, 4, 128, 64
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page)
    n, T = sum(queries), sum(queries) + 37
    q = torch.randn(T, hq * d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[n:] = float("nan")
    out = torch.full((T, hq * d), 3.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, queries[0], n], dtype=torch.int32, device=DEV)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = ops.prefill_attention_kv4(q.to(DEV), pool.to(DEV), 1, table.to(DEV), rows.to(DEV), seq, cu, max(queries), hq,
                                    hk, d, page, 0.1, out=out)
    _done()
    assert got is out and (out[n:] == 3).all()
    want, bound = oracle.attention(q[:n].double().view(n, hq, d), packed, sf, 1, table, rows, lens, queries, hq, hk, 0.1)
    _check(out[:n].view(n, hq, d), want, 1.1 * bound)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("queries", [[1, 3], [100, 30]], ids=["few", "many"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite(bad, queries, d):
    """Such a row is NaN, as by the formula; its neighbours in the same tiles are what they are."""
    lens, hq, hk, page = [300, 150], 4, 2, 32
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page)
    T = sum(queries)
    q = torch.randn(T, hq * d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    hit = torch.zeros(T, hq, dtype=torch.bool)
    for t, h, at in ((0, 1, 5), (T - 1, 3, d - 1), (T - 2, 0, 33)):
        q[t, h * d + at] = bad
        hit[t, h] = True
    cu = torch.tensor([0, queries[0], T], dtype=torch.int32, device=DEV)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = ops.prefill_attention_kv4(q.to(DEV), pool.to(DEV), 1, table.to(DEV), rows.to(DEV), seq, cu, max(queries), hq,
                                    hk, d, page, d ** -0.5).view(T, hq, d)
    _done()
    assert got[hit.to(DEV)].isnan().all()
    clean = q.double().view(T, hq, d).nan_to_num(0.0, 0.0, 0.0)
    want, bound = oracle.attention(clean, packed, sf, 1, table, rows, lens, queries, hq, hk, d ** -0.5)
    _check(got[~hit.to(DEV)], want[~hit], 1.1 * bound[~hit])


def test_one_token_of_a_large_group_with_any_stride():
    """A single row's stride says nothing, whatever it is."""
    lens, hq, d, page = [77], 100, 128, 16
    packed, sf, pool, table, rows = oracle.make_cache(lens, 1, d, page)
    q = torch.randn(1, hq * d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, [0, 1]))
    got = ops.prefill_attention_kv4(q.to(DEV).as_strided((1, hq * d), (1, 1)), pool.to(DEV), 1, table.to(DEV),
                                    rows.to(DEV), seq, cu, 1, hq, 1, d, page, 0.1)
    _done()
    want, bound = oracle.attention(q.double().view(1, hq, d), packed, sf, 1, table, rows, lens, [1], hq, 1, 0.1)
    _check(got.view(1, hq, d), want, 1.1 * bound)


def test_offsets_of_queries_that_fall_are_reported():
    pool, table, rows = (x.to(DEV) for x in oracle.make_cache([50, 40], 1, 128, 16)[2:])
    q = torch.zeros(9, 4 * 128, dtype=torch.bfloat16, device=DEV)
    seq = torch.tensor([50, 40], dtype=torch.int32, device=DEV)
    for max_q in (9, 90):  # by either path
        cu = torch.tensor([0, 9, 4], dtype=torch.int32, device=DEV)
        ops.prefill_attention_kv4(q, pool, 1, table, rows, seq, cu, max_q, 4, 1, 128, 16, 0.1)
        with pytest.raises(ops.DeviceIndexError):
            _done()


def test_offsets_beyond_32_bits():
    """The last pages of a layer of 4.5 GB: stored, read back, attended by both paths, copied."""
    hk, hq, d, page, pages = 8, 16, 128, 64, 130000
    pool = torch.zeros(2, 1, pages, hk, page * 68, dtype=torch.uint8, device=DEV)
    n = 100
    at = torch.arange(n, dtype=torch.int32, device=DEV)
    slots = at + (pages - 2) * page
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(n, hk * d, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    ops.store_kv4(k, v, pool, 0, slots, hk, d, page)
    got = [x.double().cpu() for x in ops.load_kv4(pool, 0, slots, hk, d, page)]
    for x, y in zip((k, v), got):
        c, byte = oracle.quantize(x.double().cpu().view(n, hk, d))
        assert torch.equal(y, oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte))
    table = torch.zeros(1, 128, dtype=torch.int32, device=DEV)
    table[0, :n] = slots
    row, seq, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0], [n], [0, n]))
    q = torch.randn(n, hq * d, device=DEV, generator=g).to(torch.bfloat16)
    one = ops.decode_attention_kv4(q[-1:], pool, 0, table, row, seq, hq, hk, d, page, 0.1)
    many = ops.prefill_attention_kv4(q, pool, 0, table, row, seq, cu, n, hq, hk, d, page, 0.1)
    _done()
    kk, vv = (x.repeat_interleave(hq // hk, 1) for x in got)
    sc = torch.einsum("qhd,khd->hqk", q.double().cpu().view(n, hq, d), kk) * 0.1
    p = torch.softmax(sc.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), float("-inf")), -1)
    want, a = (torch.einsum("hqk,khd->qhd", p, x) for x in (vv, vv.abs()))
    # the output's and the weights' rounding; scores of 128 products, below 2^-8 of the weights' rounding
    bound = 2.0 ** -8 * want.abs() + 1.1 * 2.0 ** -8 * a
    _check(many.view(n, hq, d), want, bound)
    _check(one.view(1, hq, d), want[-1:], bound[-1:])
    ops.copy_pages(pool, [pages - 2, pages - 1], [0, pages // 2])
    back = ops.load_kv4(pool, 0, at[:64], hk, d, page)
    assert all(torch.equal(x.double().cpu(), y[:64]) for x, y in zip(back, got))


# ----------------------------------------------------------- graphs and streams
def test_graph_replays_follow_their_buffers():
    lens, d, page, hq, hk = [700, 33, 260], 128, 16, 16, 2
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page, layers=1)
    dev = [x.to(DEV) for x in (pool, table, rows)]
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.zeros(3, hq * d, dtype=torch.bfloat16, device=DEV)
    run = lambda: ops.decode_attention_kv4(q, dev[0], 0, dev[1], dev[2], seq, hq, hk, d, page, d ** -0.5)  # noqa: E731
    run()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for now in ([700, 33, 260], [1, 20, 77], [650, 0, 5]):  # within what the table holds pages for
        x = torch.randn(3, hq * d).to(torch.bfloat16)
        q.copy_(x)
        seq.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        # both at once, each on its own stream: no scratch is shared
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        _done()
        want, bound = oracle.attention(x.double().view(3, hq, d), packed, sf, 0, table, rows, now, [1, 1, 1], hq, hk,
                                       d ** -0.5)
        for _, out in graphs:
            _check(out.view(3, hq, d), want, bound)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_graphs_replay_on_two_streams(d):
    """The many-row path captured with its plan, twice, replayed at once with other queries."""
    lens, queries, hq, hk, page = [400, 90], [130, 90], 8, 2, 64
    packed, sf, pool, table, rows = oracle.make_cache(lens, hk, d, page, layers=1)
    T = sum(queries)
    dev = [x.to(DEV) for x in (pool, table, rows)]
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, [0, 130, 220]))
    q = torch.zeros(T, hq * d, dtype=torch.bfloat16, device=DEV)
    plan = ops.KV4PrefillPlan(lens, torch.device(DEV))
    run = lambda: ops.prefill_attention_kv4(q, *dev[:1], 0, *dev[1:], seq, cu, 130, hq, hk, d, page, d ** -0.5,  # noqa: E731
                                            plan=plan)
    run()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for seed in range(2):
        x = torch.randn(T, hq * d, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
        q.copy_(x)
        torch.cuda.synchronize()
        for graph, _ in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        _done()
        want, bound = oracle.attention(x.double().view(T, hq, d), packed, sf, 0, table, rows, lens, queries, hq, hk,
                                       d ** -0.5)
        for _, out in graphs:
            _check(out.view(T, hq, d), want, 1.1 * bound)


def test_same_bits_every_time_and_on_another_stream():
    packed, sf, pool, table, rows = oracle.make_cache([3000, 5], 8, 128, 64, layers=1)
    dev = [x.to(DEV) for x in (pool, table, rows)]
    seq = torch.tensor([3000, 5], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 64 * 128, device=DEV).to(torch.bfloat16)
    run = lambda: ops.decode_attention_kv4(q, dev[0], 0, dev[1], dev[2], seq, 64, 8, 128, 64, 0.1)  # noqa: E731
    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.synchronize()
    assert torch.equal(first, again) and torch.equal(first, run())


def test_used_together():
    """A prompt, a drafted step and decode steps through store, attention and page copies."""
    hq, hk, d, page, T = 16, 4, 128, 16, 150
    g = torch.Generator().manual_seed(0)
    pages = 24
    pool = torch.zeros(2, 2, pages, hk, page * 68, dtype=torch.uint8, device=DEV)
    order = torch.randperm(pages, generator=g)[:11]
    table = torch.zeros(2, 192, dtype=torch.int32)
    at = torch.arange(11 * page)
    table[1, :11 * page] = (order[at // page] * page + at % page).to(torch.int32)
    cs = oracle.cos_sin(512, d).to(DEV)
    rows = torch.tensor([1], dtype=torch.int32, device=DEV)
    keys = []
    done = 0
    for n in (T, 3, 1, 1):
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(torch.bfloat16).to(DEV)
        pos = torch.arange(done, done + n, dtype=torch.int32, device=DEV)
        slots = table[1, done:done + n].to(DEV)
        ops.rope_store_kv4(qkv, pos, cs, None, None, pool, 1, slots, hq, hk, d, page, 1e-6)
        done += n
        keys.append(ops.load_kv4(pool, 1, slots, hk, d, page))
        seq = torch.tensor([done], dtype=torch.int32, device=DEV)
        if n == 1:
            got = ops.decode_attention_kv4(qkv, pool, 1, table.to(DEV), rows, seq, hq, hk, d, page, d ** -0.5)
        else:
            cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
            got = ops.prefill_attention_kv4(qkv, pool, 1, table.to(DEV), rows, seq, cu, n, hq, hk, d, page, d ** -0.5)
        _done()
        packed, sf = unpack_kv4(pool.cpu(), page, d)
        want, bound = oracle.attention(qkv[:, :hq * d].double().cpu().view(n, hq, d), packed, sf, 1, table, rows.cpu(),
                                       [done], [n], hq, hk, d ** -0.5)
        _check(got.view(n, hq, d), want, 1.1 * bound)
        if n == 3:  # the request moves to other pages, and its old ones are overwritten
            free = [p for p in range(pages) if p not in order.tolist()][:11]
            ops.copy_pages(pool, order, free)
            pool[:, :, order.to(DEV)] = 255
            order = torch.tensor(free)
            table[1, :11 * page] = (order[at // page] * page + at % page).to(torch.int32)
    k = torch.cat([x[0] for x in keys])
    again = ops.load_kv4(pool, 1, table[1, :done].to(DEV), hk, d, page)[0]
    assert torch.equal(k, again)


# --------------------------------------------------------------------- copies
@pytest.mark.parametrize("shape,dtype,page_dim", [
    ((2, 3, 40, 2, 16 * 68), torch.uint8, 2), ((2, 5, 33, 3, 16, 64), torch.bfloat16, 2),
    ((4, 21, 16, 72), torch.float32, 1), ((2000, 8), torch.int32, 0)])
@pytest.mark.parametrize("n", [1, 7, 10])
def test_copy_pages(shape, dtype, page_dim, n):
    g = torch.Generator().manual_seed(n)
    pool = torch.randint(0, 256, shape, generator=g).to(dtype)
    order = torch.randperm(shape[page_dim], generator=g).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]  # a page may be copied to several
    want = pool.clone()
    index = (slice(None),) * page_dim
    want[index + (torch.tensor(dst),)] = pool[index + (torch.tensor(src),)]
    dev = pool.to(DEV)
    assert ops.copy_pages(dev, src, torch.tensor(dst), page_dim) is dev
    _done()
    assert torch.equal(dev.cpu(), want)


@pytest.mark.parametrize("n", [2, 16, 17, 600])
def test_copies_that_see_one_another_are_refused(n):
    """Few pairs and many are looked over differently."""
    pool = torch.randint(0, 256, (2, 1, 1300, 1, 16 * 68), dtype=torch.uint8, device=DEV)
    before = pool.clone()
    src, dst = list(range(n)), list(range(n, 2 * n))
    for a, b in ((src, dst[:-1] + [dst[0]]), (src[:-1] + [dst[0]], dst), (src, dst[:-1] + [src[0]]), (src, dst[:-1] + [1300]),
                 (src, dst[:-1] + [-1]), (src, dst[:-1])):
        with pytest.raises((ValueError, IndexError)):
            ops.copy_pages(pool, a, b)
    _done()
    assert torch.equal(pool, before)
    ops.copy_pages(pool, tuple(src), torch.tensor(dst))
    before[:, :, dst] = before[:, :, src]
    assert torch.equal(pool, before)
    ops.copy_pages(pool, dst, dst)  # onto themselves
    assert torch.equal(pool, before)


def test_copy_many_pages():
    """More pairs than one launch takes, a page copied to itself, none at all."""
    pool = torch.randint(0, 256, (2, 2, 2100, 1, 16 * 34), dtype=torch.uint8)
    order = torch.randperm(2100).tolist()
    src, dst = order[:1033] + [order[2099]], order[1033:2066] + [order[2099]]
    want = pool.clone()
    want[:, :, dst] = pool[:, :, src]
    dev = pool.to(DEV)
    ops.copy_pages(dev, src, dst)
    ops.copy_pages(dev, [], [])
    _done()
    assert torch.equal(dev.cpu(), want)


# ------------------------------------------------------------------- refusals
def test_refusals():
    d, hk, page = 128, 2, 16
    pool = torch.zeros(2, 1, 4, hk, page * 68, dtype=torch.uint8, device=DEV)
    x = torch.zeros(3, hk * d, dtype=torch.bfloat16, device=DEV)
    i3 = torch.zeros(3, dtype=torch.int32, device=DEV)
    pt = torch.zeros(3, 64, dtype=torch.int32, device=DEV)
    q = torch.zeros(3, 4 * d, dtype=torch.bfloat16, device=DEV)
    wide = torch.zeros(3, 8 * d, dtype=torch.bfloat16, device=DEV)
    bad = [
        lambda: ops.store_kv4(x.float(), x, pool, 0, i3, hk, d, page),
        lambda: ops.store_kv4(x, x[:2], pool, 0, i3, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3[:2], hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3.long(), hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 1, i3, hk, d, page),
        lambda: ops.store_kv4(x, x, pool, 0, i3, hk, d, 32),
        lambda: ops.store_kv4(x, x, pool, 0, i3, hk, 96, page),
        lambda: ops.store_kv4(x[:, 1:], x, pool, 0, i3, 1, d, page),
        lambda: ops.store_kv4(x.cpu(), x, pool, 0, i3, hk, d, page),
        lambda: ops.load_kv4(pool, 0, i3, hk, d, page, dtype=torch.float16),
        lambda: ops.load_kv4(pool, 0, i3.cpu(), hk, d, page),
        lambda: ops.rope_store_kv4(q, i3, oracle.cos_sin(8, 64).to(DEV), None, None, pool, 0, i3, 0, hk, d, page, 1e-6),
        lambda: ops.rope_store_kv4(q, i3, oracle.cos_sin(8, d).to(DEV), x[0, :64], None, pool[:, :, :, :1].contiguous(),
                                   0, i3, 2, 1, d, page, 1e-6),
        lambda: ops.rope_store_kv4(q, i3, oracle.cos_sin(8, d).to(DEV), None, None, pool, 0, i3, 4, hk, d, page, 1e-6),
        lambda: ops.rope_store_kv4(wide, i3, oracle.cos_sin(8, 64).to(DEV), None, None, pool, 0, i3, 4, hk, d, page, 1e-6),
        lambda: ops.rope_store_kv4(wide, i3, None, None, None, pool, 0, i3, 4, hk, d, page, 1e-6),
        lambda: ops.rope_store_kv4(wide, i3, oracle.cos_sin(8, d).to(DEV), None, None, pool, 0, i3, 4, hk, d, page, 1e-6,
                                   q_out=q[:1].expand(3, -1)),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3, 3, hk, d, page, 0.1),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3, 4, hk, d, page, 0.0),
        lambda: ops.decode_attention_kv4(q, pool, 0, pt, i3, i3[:2], 4, hk, d, page, 0.1),
        lambda: ops.decode_attention_kv4(q[:2], pool, 0, pt, i3, i3, 4, hk, d, page, 0.1),
        lambda: ops.decode_attention_kv4(q.half(), pool, 0, pt, i3, i3, 4, hk, d, page, 0.1),
        lambda: ops.prefill_attention_kv4(q, pool, 0, pt, i3, i3, i3, 1, 4, hk, d, page, 0.1),
        lambda: ops.prefill_attention_kv4(q, pool, 0, pt.cpu(), i3, i3, i3, 1, 4, hk, d, page, 0.1),
        lambda: ops.copy_pages(pool, [0], i3[:1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            call()
            raise AssertionError(f"call {i} was not refused")
    _done()


def test_bad_table_entries_are_reported():
    """A page outside the pool, a request row outside the table: reported, not read."""
    d, page = 128, 16
    packed, sf, pool, table, rows = oracle.make_cache([40, 20], 1, d, page, layers=1)
    q = torch.randn(2, 8 * d, device=DEV).to(torch.bfloat16)
    seq = torch.tensor([40, 20], dtype=torch.int32, device=DEV)
    for breakage in ("slot", "row", "length"):
        t, r, n = table.clone(), rows.clone(), seq.clone()
        if breakage == "slot":
            t[r[0].item(), 16:32] = pool.shape[2] * page
        elif breakage == "row":
            r[0] = table.shape[0]
        else:
            n[0] = table.shape[1] + 1
            t[r[0].item()] = t[r[1].item(), 0].item() // page * page
        ops.decode_attention_kv4(q, pool.to(DEV), 0, t.to(DEV), r.to(DEV), n, 8, 1, d, page, 0.1)
        with pytest.raises(ops.DeviceIndexError):
            _done()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one():
    packed, sf, pool, table, rows = oracle.make_cache([300], 1, 128, 16, layers=1)
    args = [x.to("cuda:1") for x in (pool, table, rows)]
    q = torch.randn(1, 1024).to(torch.bfloat16)
    got = ops.decode_attention_kv4(q.to("cuda:1"), args[0], 0, args[1], args[2],
                                   torch.tensor([300], dtype=torch.int32, device="cuda:1"), 8, 1, 128, 16, 0.1)
    want, bound = oracle.attention(q.double().view(1, 8, 128), packed, sf, 0, table, rows, [300], [1], 8, 1, 0.1)
    _check(got.view(1, 8, 128), want, bound)


# ------------------------------------------------- many query rows: split work
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("lens,queries,hq,hk", [
    ([1300], [200], 8, 1),                            # one request over many CTAs
    ([900, 0, 40, 2000, 5], [300, 0, 40, 33, 5], 14, 2),   # groups of 7, requests without tokens or keys
    ([129, 128, 127, 256], [129, 128, 1, 200], 16, 16),    # heads of their own
    ([60] * 40, [60] * 40, 16, 4),                    # many pairs in one run
    ([500, 3, 700], [200, 9, 130], 40, 8),            # queries before the first key
    ([300], [300], 100, 1),                           # a group of 100 heads: tiles of one token
])
def test_extend_many_rows_splits(lens, queries, hq, hk, d):
    got, want, bound = _attend(lens, queries, hq, hk, d, 64, few=None)
    _check(got, want, 1.1 * bound)
