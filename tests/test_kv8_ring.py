"""How far a sequence of the 8-bit cache may be cut back (include/tsa.h, tsa_kv8): the rule that the
header states, played through on the CPU against the rows that a write keeps.

The ring holds two blocks, block i in slot i % 2.  A write keeps its rows of the last block that it
touches and the one before; the older rows of a block that it fills come from the ring.  The lowest
length a sequence may be cut back to begins as the length its own writes begin at (0, or the tokens
it took over in another's pages, whole blocks); a write up to length M raises it to
64 ((M - 1) / 64 - 1), and a cut below it, to a whole number of blocks, makes it that."""
import random

import pytest

BLOCK = 64


class Sequence:
    def __init__(self, shared=0):
        self.rows = [("theirs", i) for i in range(shared)]  # what the sequence holds
        self.pages = {i: self.rows[BLOCK * i:BLOCK * (i + 1)] for i in range(shared // BLOCK)}
        self.ring = [[None] * BLOCK, [None] * BLOCK]
        self.lowest, self.made = shared, 0

    def write(self, T):
        start, n = len(self.rows), len(self.rows) + T
        self.rows += [("own", self.made + i) for i in range(T)]
        self.made += T
        first, last = start // BLOCK, (n - 1) // BLOCK
        twin = last - (last - first) % 2  # the block that takes the first one's slot comes after it
        for blk in sorted(range(first, last + 1), key=lambda b: (b != first, b != twin)):
            p0, older = BLOCK * blk, list(self.ring[blk % 2])
            new = {r: self.rows[p0 + r] for r in range(max(start - p0, 0), min(n - p0, BLOCK))}
            if blk >= last - 1:
                for r, x in new.items():
                    self.ring[blk % 2][r] = x
            if p0 + BLOCK <= n:
                self.pages[blk] = [new.get(r, older[r]) for r in range(BLOCK)]
        self.lowest = max(self.lowest, BLOCK * (last - 1))

    def may_cut(self, n):
        return n >= self.lowest or n % BLOCK == 0

    def cut(self, n):
        self.lowest = min(self.lowest, n)
        del self.rows[n:]

    def right(self):
        full = len(self.rows) // BLOCK
        got = [x for i in range(full) for x in self.pages[i]] + self.ring[full % 2][:len(self.rows) % BLOCK]
        return got == self.rows


def test_every_cut_that_is_allowed():
    for seed in range(600):
        rng = random.Random(seed)
        s = Sequence(BLOCK * rng.choice([0, 0, 1, 2, 5]))
        for _ in range(40):
            s.write(rng.choice([1, 1, 2, 17, 63, 64, 65, 128, 129, rng.randint(1, 400)]))
            assert s.right(), seed
            for _ in range(rng.randint(0, 2)):
                n = rng.randint(0, len(s.rows)) if rng.random() < 0.5 else max(0, len(s.rows) - rng.randint(0, 130))
                if s.may_cut(n):
                    s.cut(n)
                    assert s.right(), (seed, n)


def test_rejected_drafts_are_always_allowed():
    """A cut that never falls below what was accepted, behind drafts of up to 64 tokens."""
    for seed in range(300):
        rng = random.Random(seed)
        s = Sequence(BLOCK * rng.choice([0, 1, 4]))
        s.write(rng.randint(1, 300))
        for _ in range(40):
            accepted, drafted = len(s.rows), rng.randint(1, 64)
            s.write(drafted)
            accepted += rng.randint(0, drafted)
            assert s.may_cut(accepted), (seed, accepted, s.lowest)
            s.cut(accepted)
            assert s.right(), seed


@pytest.mark.parametrize("shared,steps", [(0, [(0, 129), (65, 1), (3, 0)]), (0, [(0, 140), (76, 1), (57, 0)]), (128, [(128, 5), (123, 0)])])
def test_a_cut_below_the_lowest_length(shared, steps):
    """64 tokens or fewer behind the last write's end each time, but below the block in front of the
    longest length's, or into another sequence's block: the ring does not hold it."""
    s = Sequence(shared)
    for at, T in steps:
        allowed = s.may_cut(at)
        s.cut(at)
        if T:
            s.write(T)
    assert not allowed and not s.right()
