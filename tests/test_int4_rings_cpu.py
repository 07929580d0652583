"""The slots of the many-row 4-bit product on the CPU: its roles, barriers and
parities as they are in the kernel (minisgl/csrc/int4_gemm.cu), with copies that
land in any order. Two sets of converters take the steps in turn, so what a set
knows of a slot is what its own earlier steps told it."""

import random

import pytest

from minisgl import ops


class _Barrier:
    """An mbarrier: a phase completes when all of its arrivals (and bytes) are in; a wait by parity succeeds when the
    phase of that parity is the one before the current."""

    def __init__(self, arrivals):
        self.phase, self.need, self.left, self.copies = 0, arrivals, arrivals, 0

    def arrive(self, copies=0):
        self.copies += copies
        self.left -= 1
        self._turn()

    def landed(self):
        self.copies -= 1
        self._turn()

    def _turn(self):
        if self.left == 0 and self.copies == 0:
            self.phase, self.left = self.phase + 1, self.need

    def passed(self, parity):
        return self.phase % 2 != parity


def _run(code_slots, weight_slots, sets, steps, rng, late):
    """One CTA's steps under random delays; the first wrong read, overwritten slot or standstill as a text."""
    pfull, pempty = ([_Barrier(1) for _ in range(code_slots)] for _ in range(2))
    afull, aempty = ([_Barrier(1) for _ in range(weight_slots)] for _ in range(2))
    holds, weights, unread = [None] * code_slots, [None] * weight_slots, [None] * code_slots
    in_flight = []  # (time at which it lands, step)
    asked, read, written, issued = 0, [s for s in range(sets)], [None] * sets, 0
    mma_done = []   # commits arrive in order
    now = 0
    while issued < steps:
        now += 1
        moved = False
        for copy in [c for c in in_flight if c[0] <= now]:
            in_flight.remove(copy)
            holds[copy[1] % code_slots] = copy[1]
            pfull[copy[1] % code_slots].landed()
            moved = True
        if mma_done and mma_done[0][0] <= now:
            aempty[mma_done.pop(0)[1] % weight_slots].arrive()
            moved = True
        for role in rng.sample(range(sets + 2), sets + 2):
            if role == sets:  # the producer
                s = asked % code_slots
                if asked < steps and (asked < code_slots or pempty[s].passed((asked // code_slots - 1) & 1)):
                    if unread[s] is not None:
                        return f"step {unread[s]} was overwritten before it was read"
                    unread[s] = asked
                    pfull[s].arrive(copies=1)
                    in_flight.append((now + (rng.randint(20, 60) if rng.random() < late else rng.randint(1, 4)), asked))
                    asked += 1
                    moved = True
            elif role == sets + 1:  # the MMAs
                s = issued % weight_slots
                if afull[s].passed((issued // weight_slots) & 1):
                    if weights[s] != issued:
                        return f"the product of step {issued} took step {weights[s]}"
                    last = mma_done[-1][0] if mma_done else now
                    mma_done.append((max(last, now) + rng.randint(1, 3), issued))
                    issued += 1
                    moved = True
            else:  # a set of converters
                step = read[role]
                if written[role] is None:
                    if step < steps and pfull[step % code_slots].passed((step // code_slots) & 1):
                        if holds[step % code_slots] != step or unread[step % code_slots] != step:
                            return f"step {step} read slot {step % code_slots} while it held {holds[step % code_slots]}"
                        unread[step % code_slots] = None
                        pempty[step % code_slots].arrive()
                        written[role] = step
                        moved = True
                elif aempty[step % weight_slots].passed((step // weight_slots - 1) & 1):
                    weights[step % weight_slots] = step
                    afull[step % weight_slots].arrive()
                    written[role], read[role] = None, step + sets
                    moved = True
        if not moved and not in_flight and not mma_done:
            return f"nothing moves at step {issued}"
    return None


def _first_fault(code_slots, weight_slots, sets):
    for seed in range(400):
        rng = random.Random(seed)
        fault = _run(code_slots, weight_slots, sets, rng.choice([1, 2, 3, 7, 40]), rng, rng.choice([0.0, 0.05, 0.3]))
        if fault is not None:
            return fault
    return None


def _rings():
    if not ops.native_available():
        pytest.skip("native library not built")
    return ops.native().int4_rings()


def test_slots_of_every_tile_width():
    rings = _rings()
    assert [r[0] for r in rings] == [32, 64, 128, 192, 256]
    for rows, _, codes, weights, sets in rings:
        assert _first_fault(codes, weights, sets) is None, rows


def test_a_set_meets_only_its_own_slots():
    """With copies that land in any order a wait by parity tells a set only of fills that follow on its own."""
    for rows, _, codes, weights, sets in _rings():
        assert codes % sets == 0 and weights >= sets, rows


@pytest.mark.parametrize("slots,sets", [(3, 2), (5, 2), (4, 3)])
def test_slots_that_change_sets_are_found(slots, sets):
    """The run above finds the fault where there is one: a slot whose fills go to one set and then to another."""
    assert _first_fault(slots, 4, sets) is not None
