"""The barriers of the 8-bit product kernel (csrc/f8_mm.cu), played through on
the CPU in random orders: one thread loads stages, two issue the even and the
odd blocks' products, epilogue warps drain accumulators.  Checks that every
wait sees the phase it means (a parity wait that runs ahead by one phase would
pass at once), that products find their stage's bytes and that sums are read
from the accumulator before it is written again.

The order of the issuing threads' waits matters: an accumulator first, then
the stage.  The other order lets one of them mistake the stage's previous
phase for its own, which the second test shows."""
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0
        if self.pending == 0:
            self.phase += 1
            self.pending = self.count

    def passes(self, parity):
        """mbarrier.try_wait.parity: the phase of that parity is complete."""
        return (self.phase & 1) != parity


def play(rng, stages, bufs, halves, blocks, warps, stage_first=False):
    full, done = [Bar(1) for _ in range(stages)], [Bar(1) for _ in range(stages)]
    acc_full = [[Bar(1) for _ in range(bufs)] for _ in range(halves)]
    acc_empty = [[Bar(warps) for _ in range(bufs)] for _ in range(halves)]
    copies, products = [], [[], []]  # in flight; products of one thread complete in its order
    holds, sums = [None] * stages, {}

    def load():
        for g in range(blocks):
            s, turn = g % stages, g // stages
            while not done[s].passes((turn & 1) ^ 1):
                yield
            assert done[s].phase == turn
            holds[s] = None

            def land(s=s, g=g):
                holds[s] = g
                full[s].arrive()
            copies.append(land)
            yield

    def issue(me):
        for it in range(me, blocks, 2):
            s, buf = it % stages, it % bufs
            for h in range(halves):
                if stage_first and h == 0:
                    while not full[s].passes(it // stages & 1):
                        yield
                while not acc_empty[h][buf].passes(it // bufs & 1 ^ 1):
                    yield
                assert acc_empty[h][buf].phase == it // bufs
                if h == 0 and not stage_first:
                    while not full[s].passes(it // stages & 1):
                        yield
                assert holds[s] == it

                def finish(h=h, buf=buf, it=it, s=s):
                    assert holds[s] == it
                    sums[h, buf] = it
                    acc_full[h][buf].arrive()
                    if h == halves - 1:
                        done[s].arrive()
                products[me].append(finish)
                yield

    def drain(h):
        for g in range(blocks):
            buf = g % bufs
            while not acc_full[h][buf].passes(g // bufs & 1):
                yield
            assert acc_full[h][buf].phase == g // bufs + 1
            yield
            assert sums[h, buf] == g
            acc_empty[h][buf].arrive()
            if rng.random() < 0.05:
                for _ in range(rng.randrange(60)):
                    yield

    roles = [load(), issue(0), issue(1)] + [drain(h) for h in range(halves) for _ in range(warps)]
    for _ in range(3_000_000):
        if not roles:
            return
        x = rng.random()
        if x < 0.15 and copies:
            copies.pop(rng.randrange(len(copies)))()
        elif x < 0.3 and (products[0] or products[1]):
            k = rng.randrange(2)
            (products[k] or products[k ^ 1]).pop(0)()
        else:
            r = rng.choice(roles)
            try:
                next(r)
            except StopIteration:
                roles.remove(r)
    raise AssertionError("stuck")


SHAPES = [(5, 4, 1), (3, 2, 2), (5, 2, 2)]  # stages, accumulator buffers, halves: of f8_mm.cu's tile shapes


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_wait_means_its_own_phase(shape):
    for seed in range(60):
        rng = random.Random(seed)
        play(rng, *shape, blocks=rng.choice([1, 2, 3, 7, 20, 33]), warps=4)


def test_the_other_order_of_waits_would_not_do():
    with pytest.raises(AssertionError):
        for seed in range(200):
            play(random.Random(seed), 3, 2, 2, blocks=33, warps=4, stage_first=True)
