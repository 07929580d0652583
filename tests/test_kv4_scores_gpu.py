"""Attention over the 4-bit KV cache at scores that are large, rise or fall along the keys, or are not
finite, by the few-row and the many-row path.

Scores here are exact: queries are integers, codes are integers, scales and the softmax scale are powers of
two, and every sum of products keeps to 24 bits. So the only errors are those of the output's rounding and of
the weights' (2^-8 each, to bf16), of the polynomial (7.5e-5, twice) and of the sums over keys: the last two
within 0.1 of 2^-8. Neither grows with the scores' size: a weight is 2^(s c - m) with m taken off before the
exponential, and what m itself is rounded to cancels between a row's weights and their sum."""

import pytest
import torch

from minisgl import ops
from minisgl.quant import pack_kv4

import kv4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 2.0 ** -3


def _done():
    torch.cuda.synchronize()
    ops.check_device_errors(torch.device(DEV))


def _case(lens, queries, hq, hk, d, page, level, seed=0):
    """q, the cache and its tables: the first 32 dims of a key are the code level(position of the key, keys) at
    a scale of 8, the others random codes at a scale of 1/2; queries are an integer of the row's own in the
    first 32 dims and small ones in the others. A score in natural units: 32 q code plus a few."""
    packed, sf, _, table, rows = oracle.make_cache(lens, hk, d, page, layers=1, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    sf[0] = 20 * 8   # 1/2
    sf[0, ..., 0] = 24 * 8  # 8
    for row, n in zip(rows.tolist(), lens):
        at = table[row, :n].long()
        code = level(torch.arange(n), n) + 8
        assert ((code >= 0) & (code <= 15)).all()
        packed[0, 0, at // page, :, at % page, :16] = (code * 17).to(torch.uint8)[:, None, None]
    q = torch.randint(-2, 3, (sum(queries), hq, d), generator=g).float()
    return q, packed, sf, table, rows


def _want(q, packed, sf, table, rows, lens, queries, hq, hk, page):
    k_all, v_all = (oracle.values(packed[i, 0], sf[i, 0]) for i in range(2))
    out, size, first = [], [], 0
    for row, n, m in zip(rows.tolist(), lens, queries):
        at = table[row, :n].long()
        k, v = (x[at // page, :, at % page].repeat_interleave(hq // hk, 1) for x in (k_all, v_all))
        sc = torch.einsum("qhd,khd->hqk", q[first:first + m].double(), k) * SCALE
        assert (sc.float().double() == sc).all()
        seen = torch.arange(n)[None] <= torch.arange(n - m, n)[:, None]
        p = torch.softmax(sc.masked_fill(~seen, float("-inf")), -1)
        out.append(torch.einsum("hqk,khd->qhd", p, v))
        size.append(torch.einsum("hqk,khd->qhd", p, v.abs()))
        first += m
    out, size = torch.cat(out), torch.cat(size)
    return out, 2.0 ** -8 * out.abs() + 1.1 * 2.0 ** -8 * size


def _run(q, packed, sf, table, rows, lens, queries, page, hq, hk, d):
    T = q.shape[0]
    cu = torch.tensor([0] + list(torch.tensor(queries).cumsum(0)), dtype=torch.int32, device=DEV)
    got = ops.prefill_attention_kv4(q.to(torch.bfloat16).reshape(T, hq * d).to(DEV), pack_kv4(packed, sf).to(DEV), 0,
                                    table.to(DEV), rows.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), cu,
                                    max(queries), hq, hk, d, page, SCALE)
    _done()
    return got.view(T, hq, d)


def _check(got, want, bound):
    err = (got.double().cpu() - want).abs()
    assert (err <= bound + 1e-30).all(), f"largest error {err.max().item():.3g}, {(~(err <= bound)).double().mean():.3g} beyond"


SHAPES = [([200, 90], [150, 90], 4, 2), ([1300], [200], 8, 1), ([300], [2], 8, 2)]  # two prompts; split over CTAs; few rows


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,queries,hq,hk", SHAPES, ids=["prompts", "split", "few"])
@pytest.mark.parametrize("code", [7, -8])
def test_scores_of_any_size(lens, queries, hq, hk, d, code):
    """Rows whose scores are all near one number, from some hundreds to 2^17 in powers of two and to either
    side of zero, with half of the keys behind the mask or none."""
    case = _case(lens, queries, hq, hk, d, 16, lambda at, n: torch.full((n,), code))
    g = torch.Generator().manual_seed(7)
    base = torch.randint(1, 257, case[0].shape[:2], generator=g) * 2.0 ** torch.randint(-5, 2, case[0].shape[:2], generator=g)
    base[0, 0] = 512
    case[0][..., :32] = base[..., None]
    assert torch.equal(case[0], case[0].to(torch.bfloat16).float())
    top = (base.max() * 32 * abs(code) * 8 * SCALE).item() * 1.4427
    assert top > 2 ** 17
    got = _run(*case, lens, queries, 16, hq, hk, d)
    _check(got, *_want(*case, lens, queries, hq, hk, 16))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,queries,hq,hk", [([1950, 400], [300, 5], 8, 2), ([1950], [100], 8, 1), ([1950], [2], 8, 2)],
                         ids=["prompts", "split", "few"])
@pytest.mark.parametrize("way", [1, -1], ids=["rise", "fall"])
@pytest.mark.parametrize("base", [0.125, 0.5, 64.0])
def test_scores_that_rise_and_fall(lens, queries, hq, hk, d, way, base):
    """The scores change by 4, 16 or 2048 every 130 keys, so that with those that rise every key tile moves
    the maximum and the sums of the tiles before it are taken down."""
    case = _case(lens, queries, hq, hk, d, 64, lambda at, n: way * (at * 15 // n - 7))
    case[0][..., :32] = base
    got = _run(*case, lens, queries, 64, hq, hk, d)
    _check(got, *_want(*case, lens, queries, hq, hk, 64))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("queries", [[150, 90], [2, 1]], ids=["many", "few"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_first_tokens_that_are_not_finite(bad, queries, d):
    """A prompt's first tokens see one to six keys; with a query that is not finite their rows are NaN, as by
    the formula, and the rows beside them are what they are."""
    hq, hk, page = 4, 2, 16
    case = _case(queries, queries, hq, hk, d, page, lambda at, n: torch.full((n,), 1))
    q = case[0]
    want, bound = _want(*case, queries, queries, hq, hk, page)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool)
    for t, h, at in ((0, 0, 0), (0, 3, 40), (1, 1, 9), (2, 2, 33), (4, 0, 1), (5, 1, d - 1), (queries[0], 2, 3)):
        if t < q.shape[0]:
            q[t, h, at] = bad
            hit[t, h] = True
    got = _run(*case, queries, queries, page, hq, hk, d)
    assert got[hit.to(DEV)].isnan().all()
    _check(got[~hit.to(DEV)], want[~hit], bound[~hit])
