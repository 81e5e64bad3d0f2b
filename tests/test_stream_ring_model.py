"""CPU model of the few-token attention's stage ring (csrc/stream_attn_step.cu): one producer, four reading warps of
which `users` read a stage (warp w the stages w / users, w / users + turn, ...), full and empty barriers waited for by
parity, copies that land in any order.  Random schedules check that every read sees the stage it is meant to, that no
stage is refilled before its readers are done, and that nothing waits for ever; a ring whose slots change readers is
caught."""
import random

import pytest


class Barrier:
    """An mbarrier: `count` arrivals (and no outstanding copies) complete a phase; waits test a parity."""

    def __init__(self, count):
        self.count, self.left, self.phase, self.tx = count, count, 0, 0

    def settle(self):
        if self.left == 0 and self.tx == 0:
            self.left, self.phase = self.count, self.phase + 1

    def arrive(self, tx=0):
        self.left -= 1
        self.tx += tx
        self.settle()

    def landed(self):
        self.tx -= 1
        self.settle()

    def passed(self, parity):
        return self.phase % 2 != parity


def run(stages, ns, users, seed):
    """None if the schedule went well, else what went wrong."""
    rng = random.Random(seed)
    turn = 4 // users
    full, empty = [Barrier(1) for _ in range(ns)], [Barrier(users) for _ in range(ns)]
    holds = [None] * ns
    reads = [0] * stages
    flying = []
    produced = 0
    at = [w // users for w in range(4)]
    while True:
        moves = []
        if produced < stages and (produced < ns or empty[produced % ns].passed((produced // ns - 1) & 1)):
            moves.append(("produce",))
        moves += [("land", i) for i in range(len(flying))]
        moves += [("read", w) for w in range(4) if at[w] < stages and full[at[w] % ns].passed((at[w] // ns) & 1)]
        if not moves:
            break
        m = rng.choice(moves)
        if m[0] == "produce":
            st = produced % ns
            if produced >= ns and reads[produced - ns] < users:
                return "refilled while read"
            holds[st] = None
            full[st].arrive(tx=2)
            flying += [(st, produced), (st, produced)]
            produced += 1
        elif m[0] == "land":
            st, n = flying.pop(m[1])
            if full[st].tx == 1:
                holds[st] = n
            full[st].landed()
        else:
            w = m[1]
            st = at[w] % ns
            if holds[st] != at[w]:
                return "read a stage that had not landed"
            empty[st].arrive()
            reads[at[w]] += 1
            at[w] += turn
    if produced < stages or any(a < stages for a in at):
        return "waits for ever"
    return None


@pytest.mark.parametrize("users", [1, 2, 4])
def test_ring_of_four_slots(users):
    for seed in range(300):
        assert run(seed % 23, 4, users, seed) is None


def test_slots_that_change_readers_are_caught():
    assert any(run(20, 3, 2, seed) for seed in range(300))
    assert any(run(20, 2, 1, seed) for seed in range(300))
