"""Model check of how waveforcing_b200/csrc/paged_rows.cu shares its work (CPU).

All key tiles of all items (sequence, K/V head, tile of rows) lie in a line, of
which each CTA takes an equal stretch.  The model transcribes the arithmetic
(`find_spot`, `open_item`, `next_item`, the parts that the join reads) and runs
the lanes of a warp, which share one item in shared memory, under random
interleavings: between two warp barriers any lane may run ahead of any other.
Every lane must see the same items, the CTAs together each tile once, and the
join every part of an item.
"""
import random

import pytest

LANES = 4


def line_of(seqs, G, height, group, whole):
    """(sequence, items, tiles of an item in the line) of the sequences with items; seqs: (new tokens, key tiles)."""
    out = []
    for b, (n, tiles) in enumerate(seqs):
        items = (n * group + height - 1) // height * G if n > 0 else 0
        out.append((b, items, 1 if whole else max(tiles, 1)))
    return out


def find_spot(line, length, pos):
    first = 0
    for b, items, t in line:
        if items and first <= pos < first + items * t:
            return b, first
        first += items * t


class Warp:
    """One warp's lanes as coroutines that yield at each access to the shared item."""

    old = False  # every lane writes the item, sequence by sequence, with no barrier between its reads and that

    def __init__(self, line, length, cta, ctas, G, seed):
        self.line, self.G, self.rnd = line, G, random.Random(seed)
        self.pos = length * cta // ctas
        self.left = length * (cta + 1) // ctas - self.pos
        self.spot = find_spot(line, length, self.pos) if self.left else None
        self.it, self.seen = {}, [[] for _ in range(LANES)]

    def write(self, lane, **kv):
        if self.old or lane == 0:
            for k, v in kv.items():
                yield
                self.it[k] = v

    def read(self, k):
        yield
        return self.it[k]

    def open_from(self, lane, b):
        if self.old:
            while True:
                yield from self.write(lane, b=self.line[b][0], n=self.line[b][1], t=self.line[b][2])
                if (yield from self.read("n")):
                    return
                b = (yield from self.read("b")) + 1
        while self.line[b][1] == 0:
            b += 1
        yield "sync"
        yield from self.write(lane, b=self.line[b][0], n=self.line[b][1], t=self.line[b][2])
        yield "sync"

    def lane(self, lane):
        left = self.left
        yield from self.open_from(lane, self.spot[0])
        off, t = self.pos - self.spot[1], (yield from self.read("t"))
        item, i = off // t, off % t
        while True:
            t = yield from self.read("t")
            n = min(t - i, left)
            left -= n
            yield "sync"
            yield from self.write(lane, rt=item // self.G, hk=item % self.G, i0=i, i1=i + n)
            yield "sync"
            x = []
            for k in ("b", "rt", "hk", "i0", "i1", "t"):  # the item is worked on
                x.append((yield from self.read(k)))
            self.seen[lane].append(tuple(x))
            if left == 0:
                return
            if self.old:
                yield "sync"
            i, item = 0, item + 1
            if item == (yield from self.read("n")):
                item = 0
                yield from self.open_from(lane, (yield from self.read("b")) + 1)

    def run(self):
        lanes = [self.lane(k) for k in range(LANES)] if self.left else []
        waiting, done = set(), set()
        slow = self.rnd.randrange(LANES)
        while len(done) < len(lanes):
            k = self.rnd.choice([k for k in range(len(lanes)) if k not in waiting and k not in done])
            if k == slow and len(waiting) + len(done) < LANES - 1 and self.rnd.random() < 0.8:
                continue
            try:
                if next(lanes[k]) == "sync":
                    waiting.add(k)
            except StopIteration:
                done.add(k)
            assert not (waiting and done), "a lane has left the others at a barrier"
            if len(waiting) == LANES:
                waiting.clear()
        assert all(s == self.seen[0] for s in self.seen), "lanes of a warp disagree"
        return self.seen[0] if self.left else []


def random_line(rnd, whole):
    group, G = rnd.choice([1, 2, 4]), rnd.choice([1, 2, 3])
    seqs = [(rnd.choice([0, 0, 1, 1, 3]), rnd.choice([0, 1, 2, 5, 9])) for _ in range(rnd.randrange(1, 9))]
    height = min(max(max(n for n, _ in seqs) * group, 1), rnd.choice([1, 2, 16]))
    return line_of(seqs, G, height, group, whole), G


def run_all(seed, whole=False, kind=Warp):
    rnd = random.Random(seed)
    line, G = random_line(rnd, whole)
    length = sum(n * t for _, n, t in line)
    ctas = rnd.choice([1, 2, 3, 7, max(length, 1)])
    return line, G, length, ctas, [kind(line, length, c, ctas, G, seed * 1000 + c).run() for c in range(ctas)]


@pytest.mark.parametrize("whole", [False, True])
def test_every_tile_is_taken_once(whole):
    for seed in range(150):
        line, G, _, _, ctas = run_all(seed, whole)
        got = sorted((b, rt, hk, i) for items in ctas for b, rt, hk, i0, i1, _ in items for i in range(i0, i1))
        assert got == sorted((b, x // G, x % G, i) for b, n, t in line for x in range(n) for i in range(t))


def test_the_join_reads_every_part():
    """CTA c's last item, when begun there and not ended, has parts at c's second place and the
    first places of the next CTAs, an empty stretch's among them."""
    for seed in range(150):
        _, _, length, n_ctas, ctas = run_all(seed)
        split = {}
        for c, items in enumerate(ctas):
            for b, rt, hk, i0, i1, t in items:
                if i1 - i0 < t:
                    split.setdefault((b, rt, hk), []).append((c, 2 * c + (i0 == 0)))
        for parts in split.values():
            c = parts[0][0]
            b, rt, hk, i0, i1, t = ctas[c][-1]
            assert i0 == 0 and i1 < t
            end = length * (c + 1) // n_ctas - i1 + t
            n = (end * n_ctas + length - 1) // length - c
            places = [2 * (c + j) + (j == 0) for j in range(n)]
            empty = [2 * x for x in range(n_ctas) if not ctas[x]]  # their places hold no keys
            assert {p for _, p in parts} == set(places) - set(empty)


def test_lanes_that_write_what_others_still_read_are_caught():
    class Old(Warp):
        old = True

    with pytest.raises((AssertionError, IndexError)):
        for seed in range(150):
            run_all(seed, kind=Old)
