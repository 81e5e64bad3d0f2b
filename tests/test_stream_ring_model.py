"""CPU models of the waits of the streaming attention kernels, run under random schedules: every read sees what it is
meant to, nothing is overwritten before it is read, no copy is in flight at the end, and nothing waits for ever.

- csrc/stream_attn_tc.cu: a warp that issues loads and products and the softmax warps, around one Q, rings of K and V,
  one S (P lies over it) and one O; products run in the order of their issue, behind their issuer.
- csrc/stream_attn_step.cu: a warp's own ring, refilled by itself.
"""
import random

import pytest


class Barrier:
    """An mbarrier: `count` arrivals (and no outstanding copies) complete a phase; waits test a parity."""

    def __init__(self, count=1):
        self.count, self.left, self.phase, self.tx = count, count, 0, 0

    def settle(self):
        if self.left == 0 and self.tx == 0:
            self.left, self.phase = self.count, self.phase + 1

    def arrive(self, tx=0):
        assert self.left > 0, "an arrival too many"
        self.left -= 1
        self.tx += tx
        self.settle()

    def landed(self):
        self.tx -= 1
        self.settle()

    def passed(self, parity):
        return self.phase % 2 != parity


class Fault(Exception):
    pass


def schedule(actors, queues, seed):
    """Runs generators (each yields the (barrier, parity) it waits for) and queues of functions that run by
    themselves (`in order` or not) in random order until all are done."""
    rng = random.Random(seed)
    waits = [(a, next(a, None)) for a in actors]  # each runs up to its first wait
    waits = [(a, w) for a, w in waits if w is not None]
    while True:
        moves = [("run", i) for i, (_, (b, parity)) in enumerate(waits) if b.passed(parity)]
        for q, in_order in queues:
            moves += [("async", q, i) for i in range(min(len(q), 1) if in_order else len(q))]
        if not moves:
            if waits:
                raise Fault("waits for ever")
            return
        m = rng.choice(moves)
        if m[0] == "async":
            m[1].pop(m[2])()
        else:
            a, _ = waits[m[1]]
            w = next(a, None)
            if w is None:
                waits.pop(m[1])
            else:
                waits[m[1]] = (a, w)


def tiles(blocks, ns, seed, warps=2, v_early=False, q_early=False):
    """blocks: key blocks of each of the CTA's tiles.  v_early, q_early: mistakes that the model has to show."""
    rng = random.Random(seed ^ 12345)
    stream = [(t, j == 0) for t, n in enumerate(blocks) for j in range(n)]
    total = len(stream)
    pipe, copies = [], []
    bar_q, bar_s, bar_o, bar_p = Barrier(), Barrier(), Barrier(), Barrier(warps)
    bar_k, bar_v = [Barrier() for _ in range(ns)], [Barrier() for _ in range(ns)]
    q_mem, k_mem, v_mem = [None], [None] * ns, [None] * ns
    busy = set()  # buffers that an issued product has yet to read
    s_mem = [("done", -1)] * warps  # ("S", "P" or "done", block) of a warp's rows
    o_mem = [[] for _ in range(warps)]
    got = [[] for _ in range(warps)]

    def check(ok, what):
        if not ok:
            raise Fault(what)

    def load(name, mem, bar, at, what):
        check((name, at) not in busy, "refilled before it is read")
        mem[at] = None
        busy.add((name, at))
        bar.arrive(tx=1)
        copies.append(lambda: (mem.__setitem__(at, what), bar.landed()))

    def load_k(g):
        if g < total:
            load("k", k_mem, bar_k[g % ns], g % ns, g)

    def load_v(g):
        if g < total:
            load("v", v_mem, bar_v[g % ns], g % ns, g)

    def last(g):
        return g + 1 == total or stream[g + 1][1]

    def issue_s(g):
        def run():
            check(q_mem[0] == stream[g][0] and k_mem[g % ns] == g, "S of other rows")
            busy.discard(("k", g % ns))
            if last(g):
                busy.discard(("q", 0))
            for w in range(warps):
                check(s_mem[w] == ("done", g - 1), "S over what is not read")
                s_mem[w] = ("S", g)
            bar_s.arrive()

        pipe.append(run)

    def issue_pv(g):
        def run():
            check(v_mem[g % ns] == g, "P V of other rows")
            busy.discard(("v", g % ns))
            for w in range(warps):
                check(s_mem[w] == ("P", g), "P V before P")
                s_mem[w] = ("done", g)
                o_mem[w] = ([] if stream[g][1] else o_mem[w]) + [g]

        pipe.append(run)

    def issuer():
        if not total:
            return
        load("q", q_mem, bar_q, 0, stream[0][0])
        for g in range(ns):
            load_k(g)
            load_v(g)
        yield bar_q, 0
        yield bar_k[0], 0
        issue_s(0)
        q_phase = 1
        for g in range(total):
            more, fresh = g + 1 < total, g + 1 < total and stream[g + 1][1]
            yield bar_v[g % ns], g // ns & 1
            if more:
                yield bar_k[(g + 1) % ns], (g + 1) // ns & 1
            if q_early and fresh:
                load("q", q_mem, bar_q, 0, stream[g + 1][0])
            yield bar_p, g & 1
            issue_pv(g)
            if more and not fresh:
                issue_s(g + 1)
            else:
                pipe.append(bar_o.arrive)
                if more and not q_early:
                    load("q", q_mem, bar_q, 0, stream[g + 1][0])
            load_k(g + ns)
            if v_early:
                load_v(g + ns)
            elif g > 0:
                load_v(g - 1 + ns)
            if fresh:
                yield bar_q, q_phase & 1
                q_phase += 1
                issue_s(g + 1)
        check(not copies, "a copy is in flight at the end")

    def softmax(w):
        g = tile = 0
        for n in blocks:
            start = g
            for j in range(n):
                yield bar_s, g & 1
                check(s_mem[w] == ("S", g), "softmax of another block")
                if j > 0:  # the offset may rise: O holds all blocks before this one
                    check(o_mem[w] == list(range(start, g)), "O scaled too early or too late")
                s_mem[w] = ("P", g)
                bar_p.arrive()
                g += 1
            if n:
                yield bar_o, tile & 1
                tile += 1
                check(o_mem[w] == list(range(start, g)), "O of another tile")
                got[w].append(len(o_mem[w]))

    schedule([issuer()] + [softmax(w) for w in range(warps)], [(pipe, True), (copies, False)], seed)
    for w in range(warps):
        assert got[w] == [n for n in blocks if n]


@pytest.mark.parametrize("ns", [3, 2])  # heads up to 64 and up to 128
@pytest.mark.parametrize("blocks", [[1], [2], [7], [1, 1, 1, 1], [3, 0, 1, 5], [0, 0], [6, 2, 9], [0, 4, 0, 2, 1]])
def test_tile_protocol(ns, blocks):
    for seed in range(150):
        tiles(blocks, ns, seed)


def test_model_shows_mistakes():
    def faults(**kw):
        n = 0
        for seed in range(200):
            try:
                tiles([9, 9], 3, seed, **kw)
            except (Fault, AssertionError):
                n += 1
        return n

    assert faults() == 0
    assert faults(v_early=True) > 0  # a V stage refilled when its product is issued
    assert faults(q_early=True) > 0  # the next tile's Q loaded before the last S is known to be done


def warp_ring(items, slots, codes, seed):
    """items: copies (keys, values, keys, ...; an even number) of each item that a warp walks."""
    copies, bars = [], [Barrier() for _ in range(slots)]
    mem = [None] * slots

    def warp():
        st, parity = 0, 0

        def after(n):
            return (st + n) % slots

        for it, n_copies in enumerate(items):
            def fetch(n, to):
                if n < n_copies:
                    mem[to] = None
                    bars[to].arrive(tx=1)
                    copies.append(lambda: (mem.__setitem__(to, (it, n)), bars[to].landed()))

            def step():
                nonlocal st, parity
                st = after(1)
                parity ^= st == 0

            def read(n, at):
                if mem[at] != (it, n):
                    raise Fault("another copy's rows")

            for n in range(slots - 1):
                fetch(n, after(n))
            for n in range(0, n_copies, 2):
                fetch(n + slots - 1, after(slots - 1))
                yield bars[st], parity
                if codes:  # keys and values are held together
                    ks = st
                    step()
                    yield bars[st], parity
                    read(n, ks)
                    read(n + 1, st)
                    step()
                    fetch(n + slots, after(slots - 2))
                else:
                    read(n, st)
                    step()
                    fetch(n + slots, after(slots - 1))
                    yield bars[st], parity
                    read(n + 1, st)
                    step()
            if copies:
                raise Fault("a copy is in flight at an item's end")

    schedule([warp()], [(copies, False)], seed)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("slots", [3, 4, 5, 6, 8])
@pytest.mark.parametrize("items", [[0], [2], [4, 0, 2], [20], [14, 8, 2, 2, 30]])
def test_warp_ring(items, slots, codes):
    for seed in range(60):
        warp_ring(items, slots, codes, seed)
