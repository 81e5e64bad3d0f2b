"""CPU models of what the streaming attention kernels do when a wait runs out (csrc/stream_attn_step.cu,
csrc/stream_attn_tc.cu): whichever wait it is and whatever has landed by then, no copy is started into a slot that one is
still on its way to, nothing is written over a slot that a copy is on its way to, no warp leaves the others at a barrier, and
no copy or product is in flight when the CTA ends.

Once one wait has run out the error word is set and every other one may give up at any time; a wait that drains looks at
no error word and passes when its copy has landed or nothing is in flight any more (its limit).
"""
import random

import pytest

from test_stream_ring_model import Barrier, Fault


class Cta:
    """What is in flight, the error word and the waits of a CTA."""

    def __init__(self, seed, tired):
        self.rng, self.tired, self.err = random.Random(seed), tired, False
        self.copies, self.pipe = [], []  # land in any order; end in order

    def wait(self, bar, parity):
        """Yields until the phase is complete or the wait gives up; its value says which."""
        gives_up = self.rng.random() < self.tired
        yield lambda: bar.passed(parity) or gives_up or self.err
        ok = bar.passed(parity)
        self.err |= not ok
        return ok

    def drain(self, bar, parity, hasty=False):
        if not hasty:
            yield lambda: bar.passed(parity) or not (self.copies or self.pipe)

    def load(self, busy, at, bar):
        if at in busy:
            raise Fault("a copy into a slot that one is on its way to")
        busy.add(at)
        bar.arrive(tx=1)
        self.copies.append(lambda: (busy.discard(at), bar.landed()))

    def run(self, actors):
        waits = [(a, next(a, None)) for a in actors]
        waits = [(a, w) for a, w in waits if w is not None]
        while waits:
            moves = [("run", i) for i, (_, w) in enumerate(waits) if w()]
            moves += [("copy", i) for i in range(len(self.copies))] + [("pipe", 0)] * bool(self.pipe)
            if not moves:
                raise Fault("waits for ever")
            kind, i = self.rng.choice(moves)
            if kind != "run":
                (self.copies if kind == "copy" else self.pipe).pop(i)()
            else:
                w = next(waits[i][0], None)
                waits[i] = (waits[i][0], w)
                if w is None:
                    waits.pop(i)
        if self.copies or self.pipe:
            raise Fault("in flight at the CTA's end")


def step_group(items, slots, codes, seed, tired, warps=2, keeps_on=False, hasty=False):
    """A group of warps, each with a ring of its own; items: copies of each warp's part of an item.  keeps_on: a warp
    whose wait ran out works on as if it had not; hasty: its drain does not wait (mistakes that the model has to show)."""
    cta = Cta(seed, tired)
    joins = [Barrier(warps) for _ in range(2 * len(items))]

    def warp():
        bars, busy = [Barrier() for _ in range(slots)], set()
        st, parity, alive = 0, 0, True

        def after(n):
            return (st + n) % slots

        def step():
            nonlocal st, parity
            st = after(1)
            parity ^= st == 0

        def landed(n, sent, copies, so_far=True):
            nonlocal alive
            ok = (yield from cta.wait(bars[st], parity)) and so_far
            if not ok and not keeps_on:
                alive = False
                for i in range(n - codes, min(sent, copies)):
                    x = st + i - n
                    yield from cta.drain(bars[x % slots], parity ^ (not 0 <= x < slots), hasty)
            return alive

        for it, n_copies in enumerate(items):
            copies = n_copies if alive else 0

            def fetch(n, to):
                if n < copies:
                    cta.load(busy, to, bars[to])

            for n in range(slots - 1):
                fetch(n, after(n))
            for n in range(0, copies, 2):
                fetch(n + slots - 1, after(slots - 1))
                if codes:  # keys and values are looked at together
                    keys = yield from cta.wait(bars[st], parity)
                    step()
                    if not (yield from landed(n + 1, n + slots, copies, keys)):
                        break
                else:
                    if not (yield from landed(n, n + slots, copies)):
                        break
                    step()
                    fetch(n + slots, after(slots - 1))
                    if not (yield from landed(n + 1, n + slots + 1, copies)):
                        break
                step()
                if codes:
                    fetch(n + slots, after(slots - 2))
            if alive and busy:
                raise Fault("results over a slot that a copy is on its way to")
            for b in joins[2 * it:2 * it + 2]:  # before and after the join
                b.arrive()
                yield lambda b=b: b.phase > 0

    cta.run([warp() for _ in range(warps)])


ITEMS = [[2], [4, 0, 2], [20], [14, 8, 2, 2, 30]]


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("slots", [3, 4, 8])
@pytest.mark.parametrize("items", ITEMS)
def test_step_kernel_gives_up(items, slots, codes):
    for seed in range(80):
        step_group(items, slots, codes, seed, tired=(0.0, 0.02, 0.3)[seed % 3])


@pytest.mark.parametrize("mistake", ["keeps_on", "hasty"])
def test_step_model_shows_mistakes(mistake):
    n = 0
    for seed in range(600):
        try:
            step_group([14], 8, False, seed, 0.3, **{mistake: True})
        except (Fault, AssertionError):
            n += 1
    assert n > 0


def tiles(blocks, ns, seed, tired, warps=2, hasty=False, leaves=False):
    """A CTA of the tile kernel; blocks: key blocks of each of its tiles.  hasty: drains do not wait; leaves: a softmax
    warp that gives up does not wait for its tile's last product."""
    cta = Cta(seed, tired)
    stream = [j == 0 for n in blocks for j in range(n)]
    total = len(stream)
    bar_q, bar_s, bar_o, bar_p, bar_end = Barrier(), Barrier(), Barrier(), Barrier(warps), Barrier()
    bar_k, bar_v = [Barrier() for _ in range(ns)], [Barrier() for _ in range(ns)]
    busy = set()

    def load(name, g, bar):
        if g < total:
            cta.load(busy, (name, g % ns if name != "q" else 0), bar)

    def issuer():
        if not total:
            return
        load("q", 0, bar_q)
        for g in range(ns):
            load("k", g, bar_k[g % ns])
            load("v", g, bar_v[g % ns])
        ok = (yield from cta.wait(bar_q, 0)) and (yield from cta.wait(bar_k[0], 0))
        if ok:
            cta.pipe.append(bar_s.arrive)
        q_phase, g = 1, 0
        while ok and g < total:
            more, fresh = g + 1 < total, g + 1 < total and stream[g + 1]
            ok = yield from cta.wait(bar_v[g % ns], g // ns & 1)
            if ok and more:
                ok = yield from cta.wait(bar_k[(g + 1) % ns], (g + 1) // ns & 1)
            ok = ok and (yield from cta.wait(bar_p, g & 1))
            if not ok:
                break
            cta.pipe.append(lambda: None)  # P V
            if more and not fresh:
                cta.pipe.append(bar_s.arrive)
            else:
                cta.pipe.append(bar_o.arrive)
                if more:
                    load("q", 0, bar_q)
            load("k", g + ns, bar_k[g % ns])
            if g > 0:
                load("v", g - 1 + ns, bar_v[(g - 1) % ns])
            if fresh:
                ok = yield from cta.wait(bar_q, q_phase & 1)
                if not ok:
                    break
                q_phase += 1
                cta.pipe.append(bar_s.arrive)
            g += 1
        if not ok:
            cta.pipe.append(bar_end.arrive)
            yield from cta.drain(bar_end, 0, hasty)
            for parity in (0, 1):
                for b in [bar_q] + bar_k + bar_v:
                    yield from cta.drain(b, parity, hasty)

    def softmax():
        g = tile = 0
        ok = True
        for n in blocks:
            for _ in range(n):
                ok = yield from cta.wait(bar_s, g & 1)
                if not ok:
                    break
                bar_p.arrive()
                g += 1
            if ok and n:
                ok = yield from cta.wait(bar_o, tile & 1)
                tile += ok
            if not ok:
                break
        if not ok and not leaves:
            yield from cta.drain(bar_o, tile & 1, hasty)

    cta.run([issuer()] + [softmax() for _ in range(warps)])


@pytest.mark.parametrize("ns", [3, 2])
@pytest.mark.parametrize("blocks", [[1], [7], [1, 1, 1, 1], [3, 0, 1, 5], [0, 0], [6, 2, 9]])
def test_tile_kernel_gives_up(ns, blocks):
    for seed in range(120):
        tiles(blocks, ns, seed, tired=(0.0, 0.02, 0.2)[seed % 3])


@pytest.mark.parametrize("mistake", ["hasty", "leaves"])
def test_tile_model_shows_mistakes(mistake):
    n = 0
    for seed in range(600):
        try:
            tiles([2, 3], 3, seed, 0.1, **{mistake: True})
        except (Fault, AssertionError):
            n += 1
    assert n > 0
