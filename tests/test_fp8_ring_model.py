"""A model of the wide 8-bit product kernel's barriers (csrc/gemm_fp8.cu): its
warps as generators, stepped in random order, with parity waits answered as an
mbarrier answers them and loads that land in any order.  It holds the kernel's
rings sound, and shows that over an odd number of slots two issuers have to take
turns at the wait for a load."""
import os
import random
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Bar:
    def __init__(self, count):
        self.count, self.pending, self.phase = count, 0, 0

    def arrive(self):
        self.pending += 1
        assert self.pending <= self.count, "too many arrivals"
        if self.pending == self.count:
            self.pending, self.phase = 0, self.phase + 1

    def passed(self, parity):  # a wait for the phase of this parity returns
        return (self.phase & 1) != parity


def simulate(sets, slots, blocks, tiles, seed, turns=True):
    rnd = random.Random(seed)
    full, empty = [Bar(1) for _ in range(slots)], [Bar(1) for _ in range(slots)]
    tfull, tempty = [Bar(2) for _ in range(2 * sets)], [Bar(1) for _ in range(2 * sets)]
    turn = [Bar(1), Bar(1)]
    ring, acc, scales = [None] * slots, [None] * (2 * sets), [None] * (2 * sets)
    queue, flying, drained, loaded = [], [], [], []

    def order():  # (ring index, set, block of the set, what it is)
        i, js = 0, [0, 0]
        for t in range(tiles):
            s = t % sets
            for b in range(blocks):
                yield i, s, js[s], (t, b)
                i, js[s] = i + 1, js[s] + 1

    def load():
        for i, _, _, what in order():
            while not empty[i % slots].passed((i // slots & 1) ^ 1):
                yield
            ring[i % slots] = None
            flying.append((i % slots, what))
            yield
        loaded.append(True)

    def land():
        while not (loaded and not flying):
            if flying:
                s, what = flying.pop(rnd.randrange(len(flying)))
                ring[s] = what
                full[s].arrive()
            yield

    def issue(e):
        for i, s, j, what in order():
            if i & 1 == e:
                while turns and not turn[e].passed((i >> 1 & 1) ^ e ^ 1):
                    yield
                while not full[i % slots].passed(i // slots & 1):
                    yield
                turn[e ^ 1].arrive()
                yield
                buf = 2 * s + (j & 1)
                while not tempty[buf].passed((j >> 1 & 1) ^ 1):
                    yield
                queue.append((i % slots, buf, what))
                yield

    def tensor():
        for _ in range(tiles * blocks):
            while not queue:
                yield
            slot, buf, what = queue.pop(0)
            assert ring[slot] == what, "multiplied what had not landed"
            acc[buf] = what
            yield
            empty[slot].arrive()
            tfull[buf].arrive()

    def scale():
        for _, s, j, what in order():
            buf = 2 * s + (j & 1)
            while not tempty[buf].passed((j >> 1 & 1) ^ 1):
                yield
            scales[buf] = what
            yield
            tfull[buf].arrive()

    def drain(mine):
        for _, s, j, what in order():
            if s == mine:
                buf = 2 * s + (j & 1)
                while not tfull[buf].passed(j >> 1 & 1):
                    yield
                assert acc[buf] == what and scales[buf] == what, "drained another block"
                yield
                tempty[buf].arrive()
                drained.append(what)
                for _ in range(rnd.randrange(30) if what[1] == blocks - 1 else 0):  # the epilogue
                    yield

    actors = [load(), land(), tensor(), scale()] + [issue(e) for e in range(2)] + [drain(s) for s in range(sets)]
    weights, steps = None, 0
    while actors:
        if weights is None or rnd.random() < 0.01:
            weights = [10 ** rnd.uniform(-3, 0) for _ in actors]
        k = rnd.choices(range(len(actors)), weights)[0]
        steps += 1
        assert steps < 400000, "stuck"
        try:
            next(actors[k])
        except StopIteration:
            del actors[k], weights[k]
    assert len(drained) == tiles * blocks


def kernel_configurations():
    """(sets, slots) of the 256- and 128-column tiles, from the source."""
    src = open(os.path.join(ROOT, "onnx_b200", "csrc", "gemm_fp8.cu")).read()
    assert "TURNS = S % 2 != 0;" in src
    m = re.search(r"static constexpr int S = BN == 256 \? (\d+) : (\d+);", src)
    return [(256 // bn, int(s)) for bn, s in ((256, m.group(1)), (128, m.group(2)))]


@pytest.mark.parametrize("sets, slots", kernel_configurations())
@pytest.mark.parametrize("blocks", [1, 2, 3, 4, 5, 7])
def test_rings_are_sound(sets, slots, blocks):
    for tiles in (1, 2, 7):
        for seed in range(12):
            simulate(sets, slots, blocks, tiles, seed, turns=slots % 2 != 0)


def test_issuers_of_an_odd_ring_take_turns():
    def fails(slots, turns):
        n = 0
        for seed in range(60):
            try:
                simulate(2, slots, 3, 13, seed, turns)
            except AssertionError:
                n += 1
        return n
    assert fails(3, False) and not fails(3, True) and not fails(4, False)
