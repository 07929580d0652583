"""Lengths, offsets and plans on the device that the host cannot check: attention over the 4-bit KV cache reports
them and reads nothing outside its tensors."""

import pytest
import torch

from minisgl import ops

import kv4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _done():
    torch.cuda.synchronize()
    ops.check_device_errors(torch.device(DEV))


def _reported():
    with pytest.raises(ops.DeviceIndexError):
        _done()


class _Batch:
    """Requests of `lens` keys and `queries` tokens, and what attention over them gives."""

    def __init__(self, lens, queries, hq=8, hk=2, d=128, page=16):
        self.lens, self.queries, self.heads = lens, queries, (hq, hk, d, page)
        self.packed, self.sf, pool, table, rows = oracle.make_cache(lens, hk, d, page, layers=1)
        self.table, self.rows = table, rows
        self.pool, self.pt, self.rr = pool.to(DEV), table.to(DEV), rows.to(DEV)
        self.cu = [0]
        for n in queries:
            self.cu.append(self.cu[-1] + n)
        self.q = torch.randn(self.cu[-1], hq * d, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)

    def run(self, lens=None, cu=None, plan=None, out=None):
        hq, hk, d, page = self.heads
        seq = torch.tensor(self.lens if lens is None else lens, dtype=torch.int32, device=DEV)
        cu = torch.tensor(self.cu if cu is None else cu, dtype=torch.int32, device=DEV)
        return ops.prefill_attention_kv4(self.q.to(DEV), self.pool, 0, self.pt, self.rr, seq, cu, max(self.queries), hq,
                                         hk, d, page, d ** -0.5, plan=plan, out=out).view(-1, hq, d)

    def check(self, got, request, lens=None):
        """The rows of one request, with as many keys as `lens` says."""
        hq, hk, d, _ = self.heads
        lo, hi = self.cu[request], self.cu[request + 1]
        n = (lens or self.lens)[request]
        want, bound = oracle.attention(self.q[lo:hi].double().view(-1, hq, d), self.packed, self.sf, 0, self.table,
                                       self.rows[request:request + 1], [n], [hi - lo], hq, hk, d ** -0.5)
        assert ((got[lo:hi].double().cpu() - want).abs() <= 1.1 * bound + 1e-30).all()


@pytest.mark.parametrize("queries", [[150, 90, 30], [3, 2, 1]], ids=["many", "few"])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 100000])
def test_lengths_beyond_the_table(queries, length):
    batch = _Batch([300, 200, 90], queries)
    for at in range(3):
        lens = list(batch.lens)
        lens[at] = length
        plan = ops.KV4PrefillPlan(batch.lens, torch.device(DEV)) if queries[0] > 3 else None
        got = batch.run(lens, plan=plan)
        _reported()
        for other in range(3):
            if other != at:
                batch.check(got, other)
    if queries[0] > 3:  # the host makes no plan of such lengths
        with pytest.raises(ValueError, match="positions"):
            batch.run(lens)


@pytest.mark.parametrize("queries", [[150, 90, 30], [3, 2, 1]], ids=["many", "few"])
def test_negative_lengths_are_no_keys(queries):
    batch = _Batch([300, 200, 90], queries)
    plan = ops.KV4PrefillPlan(batch.lens, torch.device(DEV)) if queries[0] > 3 else None
    for length in (-1, -2 ** 31):
        got = batch.run([300, length, 90], plan=plan)
        _done()
        assert (got[batch.cu[1]:batch.cu[2]] == 0).all()
        batch.check(got, 0), batch.check(got, 2)


@pytest.mark.parametrize("queries", [[150, 90, 30], [3, 2, 1]], ids=["many", "few"])
def test_offsets_that_fall_leave_no_work(queries):
    """Rows of several requests at once would add up to more tiles than a call counts."""
    batch = _Batch([300, 200, 90], queries)
    T = batch.cu[-1]
    plan = ops.KV4PrefillPlan(batch.lens, torch.device(DEV)) if queries[0] > 3 else None
    for cu in ([0, T, 0, T], [0, T, T - 1, T], [0, 2, T, -4]):
        out = torch.full((T, 8 * 128), 3.0, dtype=torch.bfloat16, device=DEV)
        batch.run(cu=cu, plan=plan, out=out)
        _reported()
        assert (out == 3).all()
    got = batch.run(plan=plan)
    _done()
    for request in range(3):
        batch.check(got, request)


@pytest.mark.parametrize("planned", [[300, 200, 90], [200, 200, 200], [310, 150, 90], [305, 200, 80], [90, 200, 310]],
                         ids=lambda x: "-".join(map(str, x)))
def test_a_plan_of_fewer_keys_than_a_request_has(planned):
    """Growth within a tile, beyond one, of any request: reported, the request's rows zeros, the others' right.
    A plan may hold more keys than a request has."""
    lens = [310, 200, 90]
    batch = _Batch(lens, [150, 90, 30])
    got = batch.run(plan=ops.KV4PrefillPlan(planned, torch.device(DEV)))
    _reported()
    for request, (n, m) in enumerate(zip(lens, planned)):
        if n <= m:
            batch.check(got, request)
        else:
            assert (got[batch.cu[request]:batch.cu[request + 1]] == 0).all()
    for now in ([310, 200, 90], [7, 129, 128], [256, 0, 1]):
        got = batch.run(now, plan=ops.KV4PrefillPlan([310, 200, 130], torch.device(DEV)))
        _done()
        for request in range(3):
            batch.check(got, request, now)


@pytest.mark.parametrize("max_q", [200, 1], ids=["many", "few"])
def test_a_batch_of_no_requests(max_q):
    hq, hk, d, page = 8, 2, 128, 16
    pool = torch.zeros(2, 1, 4, hk, page * 68, dtype=torch.uint8, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    table, cu = torch.zeros(1, 64, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, hq * d, dtype=torch.bfloat16, device=DEV)
    got = ops.prefill_attention_kv4(q, pool, 0, table, none, none, cu, max_q, hq, hk, d, page, 0.1)
    _done()
    assert got.shape == (0, hq * d)


@pytest.mark.parametrize("rows,tiles,max_q", [(16383, 131078, 1), (16383, 131078, 100)], ids=["few", "many"])
def test_more_tiles_than_32_bits_count(rows, tiles, max_q):
    """A unit of query rows (8 of them, or 256) may have a tile for each 128 positions of the table, the last
    one begun, and two for what it costs beside them. The call with one tile too many is refused, the one
    before it runs."""
    d, page = 64, 16
    T = (rows - 1) * (8 if max_q == 1 else 256)
    assert rows * (2 + tiles) <= 2 ** 31 - 1 < rows * (2 + tiles + 1)
    pool = torch.zeros(2, 1, 4, 1, page * 34, dtype=torch.uint8, device=DEV)
    row, seq, cu = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0], [5], [0, T]))
    q = torch.zeros(1, d, dtype=torch.bfloat16, device=DEV).expand(T, -1)
    table = torch.zeros(tiles * 128 + 1, dtype=torch.int32, device=DEV)
    call = lambda n: ops.prefill_attention_kv4(q, pool, 0, table[:n].view(1, n), row, seq, cu, max_q, 1, 1, d, page, 0.1)  # noqa: E731
    with pytest.raises(RuntimeError, match="too many tiles"):
        call(tiles * 128 + 1)
    out = call(tiles * 128)
    _done()
    # rows before the first key are zeros; a pool of zero bytes holds -8 at a scale of 2^-21 everywhere
    assert (out[:-5] == 0).all() and (out[-5:] == -2.0 ** -18).all()


def test_a_captured_prompt_with_shorter_lengths():
    """A plan holds the keys of the capture; replays with fewer keys read nothing of the table behind them,
    where entries are of no page."""
    lens = [400, 200, 90]
    batch = _Batch(lens, [150, 90, 30])
    hq, hk, d, page = batch.heads
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu = torch.tensor(batch.cu, dtype=torch.int32, device=DEV)
    q, plan = batch.q.to(DEV), ops.KV4PrefillPlan(lens, torch.device(DEV))
    call = lambda: ops.prefill_attention_kv4(q, batch.pool, 0, batch.pt, batch.rr, seq, cu, 150, hq, hk, d, page,  # noqa: E731
                                             d ** -0.5, plan=plan)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for now in ([400, 200, 90], [150, 100, 31], [300, 0, 1], [129, 128, 90]):
        seq.copy_(torch.tensor(now, dtype=torch.int32))
        for row, n in zip(batch.rows.tolist(), now):
            batch.pt[row, n:] = -1 if n % 2 else 2 ** 31 - 1
            batch.pt[row, :n] = batch.table[row, :n].to(DEV)
        graph.replay()
        _done()
        for request in range(3):
            batch.check(out.view(-1, hq, d), request, now)


@pytest.mark.parametrize("queries", [[150, 90, 30], [3, 2, 1]], ids=["many", "few"])
def test_same_bits_every_time(queries):
    """Records of split work are joined in the order of their runs, so calls repeat bit for bit."""
    batch = _Batch([2000, 900, 90], queries)
    first = batch.run()
    torch.cuda.synchronize()
    for _ in range(5):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            again = batch.run()
        torch.cuda.synchronize()
        assert torch.equal(first, again)
    _done()
