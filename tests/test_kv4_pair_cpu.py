"""The meetings of the two warps that share rows of scores in the many-row kernel of the 4-bit KV cache, on the
CPU: the control flow of both as it is in the kernel (minisgl/csrc/kv4_prefill.cu), with bounded waits that run
out at any place for one of them, the other or both. Neither may stand at the barrier alone, since no time
limit ends that on a GPU."""

import os
import re

import pytest

KERNEL = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minisgl", "csrc", "kv4_prefill.cu")


class _Waits:
    """Bounded waits of one warp: number `fails` runs out (None: none does), those after it too if `stays`."""

    def __init__(self, fails, stays):
        self.count, self.fails, self.stays = 0, fails, stays

    def __call__(self):
        i, self.count = self.count, self.count + 1
        return self.fails is None or not (i == self.fails or (self.stays and i > self.fails))


def _warp(pieces, wait, log):
    """A warp of the pair; yields at every meeting what it says there and is sent what both say."""
    ok, k = True, 0
    while (yield ok and wait() and k < len(pieces)):  # the next piece's description
        for _ in range(pieces[k]):
            if ok:
                ok = wait()  # for the tile's scores
            yield True       # maxima swapped
        if ok and pieces[k] > 0:
            ok = wait()      # for the output
        yield True
        yield True           # sums swapped
        log.append((k, ok))
        k += 1


def _warp_alone(pieces, wait, log):
    """The same with loops that each warp leaves by its own waits."""
    ok, k = True, 0
    while ok and wait() and k < len(pieces):
        done = 0
        while ok and done < pieces[k]:
            ok = wait()
            yield True
            done += 1
        if ok and pieces[k] > 0:
            ok = wait()
        for _ in range(4):
            yield True
        log.append((k, ok))
        k += 1


def _stands(form, pieces, fails, stays):
    """Whether one warp waits at a meeting that the other never comes to; and what each wrote."""
    logs = [], []
    warps = [form(pieces, _Waits(f, stays), log) for f, log in zip(fails, logs)]
    said = [next(w, None) for w in warps]
    while None not in said:
        both = all(said)
        said = []
        for w in warps:
            try:
                said.append(w.send(both))
            except StopIteration:
                said.append(None)
    return said != [None, None], logs


RUNS = [[2, 0, 3], [1], [], [0, 0], [4, 1]]


def _all(form):
    for pieces in RUNS:
        places = [None, *range(1 + sum(1 + n + (n > 0) for n in pieces))]
        for a in places:
            for b in places:
                for stays in (False, True):
                    yield pieces, (a, b), _stands(form, pieces, (a, b), stays)


def test_no_warp_stands_alone_whichever_wait_runs_out():
    for pieces, fails, (stands, logs) in _all(_warp):
        assert not stands, (pieces, fails)
        assert [k for k, _ in logs[0]] == [k for k, _ in logs[1]]
        if fails == (None, None):
            assert logs[0] == logs[1] == [(k, True) for k in range(len(pieces))]


def test_the_check_sees_a_warp_that_stands_alone():
    assert any(stands for _, _, (stands, _) in _all(_warp_alone))
    assert not any(stands for _, fails, (stands, _) in _all(_warp_alone) if fails == (None, None))


@pytest.fixture(scope="module")
def softmax():
    with open(KERNEL, encoding="utf-8") as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    begin = text.index("auto agree = [&]")
    return text[begin:text.index("atomicExch(s_abort, 1)", begin)]


def test_the_kernel_has_the_control_flow_of_the_check(softmax):
    """Its meetings: the head of the loop over pieces, one in every tile, two after them; no way out between."""
    loops = re.findall(r"for \(int [kj] = 0; ([^;]*);", softmax)
    assert loops[0] == "agree(ok && __all_sync(0xffffffffu, describe(k)))" and loops[1] == "j < nx"
    body = softmax[softmax.index("for (int k = 0; agree"):]
    assert softmax.count("agree(") == 1 and body.count("pair_sync();") == 3
    assert not re.search(r"\b(break|return|continue|goto)\b", body)
    tile = body[body.index("for (int j = 0; j < nx"):body.index("wait_asleep(&o_done")]
    assert tile.count("pair_sync();") == 1
    # no meeting under a condition: each is a statement at the loops' own depth
    assert re.findall(r"\n( *)pair_sync\(\);", body) == [" " * 8, " " * 6, " " * 6]
