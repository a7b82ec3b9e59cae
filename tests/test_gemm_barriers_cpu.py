"""The barriers of the GEMM kernels that dequantise inside, as a model on the CPU.

A stage of the ring is filled by a producer, dequantised by one of the sets of warps that deal the k-steps out among
themselves, and read by the MMAs, which free it.  ``mbarrier.try_wait.parity`` tells only whether the phase under way
has another parity than the one asked for.  A waiter that sees every phase, or one whose phase before is known to be
over, gets the right answer; one that sees every second phase does not, where the copies of one stage land later than
those of the next ones.  The model runs the roles with random delays and checks that every k-step is dequantised
from its own words and multiplied with its own tile.  Numbers of stages, sets and barriers are read from the sources.
"""
import heapq
import os
import random
import re

import pytest

import __graft_entry__

SOURCE = os.path.join(__graft_entry__.PKG_DIR, "csrc", "awq_gemm.cu")


class Barrier:
    def __init__(self, count):
        self.count, self.phase, self.pending, self.tx = count, 0, count, 0

    def arrive(self, tx=0):
        self.pending -= 1
        self.tx += tx
        self._flip()

    def complete(self, n=1):
        self.tx -= n
        self._flip()

    def _flip(self):
        assert self.pending >= 0, "more arrivals than a phase takes"
        if self.pending == 0 and self.tx == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def passes(self, parity):
        return (self.phase & 1) != parity


class Fault(Exception):
    pass


def simulate(stages, sets, ctas, fulls, steps, seed):
    """Runs the roles, with ``fulls`` barriers of landed copies; raises Fault where a step meets another step's data, or where all of them wait for good."""
    rng = random.Random(seed)
    slow = rng.randrange(steps)                  # one copy lands late
    full = [[Barrier(1) for _ in range(fulls)] for _ in range(ctas)]
    empty = [[Barrier(1) for _ in range(stages)] for _ in range(ctas)]
    afull = [Barrier(ctas) for _ in range(stages)]
    words = [[None] * stages for _ in range(ctas)]
    tile = [[None] * stages for _ in range(ctas)]
    events, order = [], 0

    def later(delay, what):
        nonlocal order
        order += 1
        heapq.heappush(events, (now + delay, order, what))

    def producer(cta):
        for it in range(steps):
            s = it % stages
            if it >= stages:
                yield lambda: empty[cta][s].passes(((it // stages) & 1) ^ 1)
            full[cta][it % fulls].arrive(tx=1)

            def land(it=it, s=s):
                words[cta][s] = it
                full[cta][it % fulls].complete()
            later(rng.uniform(5, 10) * (8 if it == slow else 1), land)

    def dequant(cta, mine):
        for it in range(mine, steps, sets):
            s = it % stages
            yield lambda: full[cta][it % fulls].passes((it // fulls) & 1)
            if words[cta][s] != it:
                raise Fault(f"step {it} dequantises the words of step {words[cta][s]}")
            yield now + rng.uniform(0.5, 2)
            tile[cta][s] = it
            afull[s].arrive()

    def mma():
        last = 0.0
        for it in range(steps):
            s = it % stages
            yield lambda: afull[s].passes((it // stages) & 1)
            if any(t[s] != it for t in tile):
                raise Fault(f"step {it} multiplies the tiles {[t[s] for t in tile]}")
            last = max(last, now) + rng.uniform(0.5, 2)

            def done(s=s, it=it):
                if any(t[s] != it for t in tile):
                    raise Fault(f"the tile of step {it} is overwritten while it is read")
                for e in empty:
                    e[s].arrive()
            later(last - now, done)

    now = 0.0
    waiting = []
    for role in [producer(c) for c in range(ctas)] + [dequant(c, g) for c in range(ctas) for g in range(sets)] + [mma()]:
        waiting.append([role, None])
    while waiting:
        moved = True
        while moved:
            moved = False
            for entry in list(waiting):
                want = entry[1]
                if want is not None and (not want() if callable(want) else now < want):
                    continue
                moved = True
                try:
                    entry[1] = next(entry[0])
                    if not callable(entry[1]):
                        later(entry[1] - now, lambda: None)
                except StopIteration:
                    waiting.remove(entry)
        if not waiting:
            return
        if not events:
            raise Fault("every role waits for good")
        now, _, what = heapq.heappop(events)
        what()


def test_the_model_sees_a_set_that_skips_phases():
    """Five stages dealt to two sets, with one barrier for each stage."""
    faults = 0
    for seed in range(200):
        try:
            simulate(5, 2, 2, 5, 24, seed)
        except (Fault, AssertionError):
            faults += 1
    assert faults > 20


@pytest.mark.parametrize("ctas", [1, 2])
def test_pair_kernel(ctas):
    text = open(SOURCE).read()
    sets = int(re.search(r"int SETS = PANEL \? 0 : (\d+);", text)[1])
    stages = int(re.search(r"int SST = PANEL \? \d+ : (\d+);", text)[1])
    each_set = re.search(r"int FST = PANEL \? SST : SETS \* SST;", text) and "&full_w[f], (it / FST) & 1" in text
    for seed in range(400):
        simulate(stages, sets, ctas, sets * stages if each_set else stages, 40, seed)


def test_persistent_kernel():
    """A set of the persistent kernel always meets the same stages, so it sees all of their phases."""
    text = open(SOURCE).read()
    found = set(re.findall(r"launch_gemm_persistent<\d+, (\d+), (\d+), EPI, (\d+)>", text))
    assert found
    for stages, slots, sets in ((int(a), int(b), int(c)) for a, b, c in found):
        assert stages % sets == 0 and slots % sets == 0
        for seed in range(200):
            simulate(stages, sets, 1, stages, 40, seed)
