"""The shared-memory ring of the chunk attention's tensor-core kernel
(attn_chunk_tc_kernel, gb_chunk.cu) when a wait runs out, modelled on the CPU:
two loaders bring K and V tiles by asynchronous copies whose bytes a barrier
counts, a third warp zeroes what lies behind a sequence's end and reports that
tile full, the products read tiles and report them empty when they have ended.

A barrier here is an mbarrier: arrivals outstanding in its phase, and bytes
expected. An arrival in a phase that has none outstanding (all have come, bytes
still on their way) is undefined, and so is a copy that lands after the block
has ended. The model gives any wait up at random and checks that neither
happens where the fetching warps start no more copies once they see that a wait
has run out, although the products go on and report slots empty, and that the
first happens where they go on too."""
import random

import pytest


class Undefined(Exception):
    pass


class Barrier:
    def __init__(self):
        self.out, self.bytes, self.phases = 1, 0, 0

    def turn(self):
        if self.out == 0 and self.bytes == 0:
            self.phases += 1
            self.out = 1

    def arrive(self, expect=0):
        if self.out == 0:
            raise Undefined("an arrival in a phase that has all of its own")
        self.out -= 1
        self.bytes += expect
        self.turn()

    def landed(self):
        self.bytes -= 1
        self.turn()

    def done(self, parity):
        return self.phases & 1 != parity


class Block:
    def __init__(self, pieces, NS, seed, give_up, stops):
        self.NS = NS  # slots: 5 at head_dim 128, 10 at 64
        self.r, self.give_up, self.stops, self.dead = random.Random(seed), give_up, stops, False
        self.pieces = pieces  # (tiles, whether the last of them is the sequence's end)
        self.full, self.empty, self.ended = ([Barrier() for _ in range(NS)] for _ in range(3))
        self.fetched = [None, None]
        self.haste = self.r.choice([1.0, 0.1, 0.01])  # of the copies
        self.flight, self.queue = [], []  # copies on their way; products' reports

    def wait(self, bar, parity):
        """Yields until the phase is over: True; False where it gives up or another wait has."""
        while not bar.done(parity):
            if self.dead:
                return False
            if self.r.random() < self.give_up:
                self.dead = True
                return False
            yield
        return True

    def tiles(self):
        for n, end in self.pieces:
            for t in range(n):
                yield end and t + 1 == n

    def loader(self, kv):
        NS = self.NS
        n, last = 0, {}
        phase = [0] * NS
        self.fetched[kv] = None
        for end in self.tiles():
            slot, lap = (n + kv) % NS, (n + kv) // NS
            got = yield from self.wait(self.empty[slot], lap & 1 ^ 1)
            if self.stops and (self.dead or not got):
                break
            bar = self.ended[slot] if kv and end else self.full[slot]
            bar.arrive(expect=1)
            self.flight.append(bar)
            if kv and end:
                last[n + 1] = (bar, phase[slot])
                phase[slot] ^= 1
            else:
                last[n + kv] = (bar, lap & 1)
            n += 2
            yield
        self.fetched[kv] = n
        while self.fetched[kv ^ 1] is None:
            yield
        for i in range(max(0, n - NS - 1), n):  # the last waits are made all the same
            if i & 1 == kv and not i + NS < self.fetched[(i + NS) & 1]:
                bar, parity = last[i]
                for k in range(4000):
                    if bar.done(parity):
                        break
                    yield
                else:
                    raise Undefined("a last wait for nothing")

    def zeros(self):
        NS = self.NS
        n, phase = 0, [0] * NS
        for end in self.tiles():
            if end:
                slot = (n + 1) % NS
                got = yield from self.wait(self.ended[slot], phase[slot])
                if self.stops and (self.dead or not got):
                    return
                phase[slot] ^= 1
                self.full[slot].arrive()
            n += 2
            yield

    def products(self):
        NS = self.NS
        n = 0
        for _ in self.tiles():
            for i in (n, n + 1):
                yield from self.wait(self.full[i % NS], i // NS & 1)
                self.queue.append(self.empty[i % NS])
            n += 2
            yield
        while self.queue:
            yield

    def run(self):
        actors = [self.loader(0), self.loader(1), self.zeros(), self.products()]
        for _ in range(200000):
            if not actors:
                break
            pick = self.r.randrange(len(actors) + 2)
            if pick < len(actors):
                try:
                    next(actors[pick])
                except StopIteration:
                    del actors[pick]
            elif self.flight and pick == len(actors):
                if self.r.random() < self.haste:
                    self.flight.pop(self.r.randrange(len(self.flight))).landed()
            elif self.queue:
                self.queue.pop(0).arrive()  # products end in order
        assert not actors
        if self.flight:
            raise Undefined("a copy lands after the end")
        return self.dead


def blocks(give_up, stops, count):
    for seed in range(count):
        r = random.Random(seed)
        pieces = [(r.randint(1, 9), r.random() < 0.5) for _ in range(r.randint(1, 6))]
        yield Block(pieces, r.choice([5, 10]), seed, give_up, stops)


def test_no_wait_runs_out():
    for b in blocks(0.0, True, 200):
        assert not b.run()


@pytest.mark.parametrize("give_up", [0.001, 0.01, 0.1, 1.0])
def test_a_wait_that_runs_out_leaves_nothing_on_its_way(give_up):
    dead = sum(b.run() for b in blocks(give_up, True, 400))
    assert dead > 40


def test_going_on_would_not_do():
    undefined = 0
    for b in blocks(0.01, False, 400):
        try:
            b.run()
        except Undefined:
            undefined += 1
    assert undefined > 40
