"""Model check of the synchronisation of waveforcing_b200/csrc/paged_tile.cu (CPU).

The kernel's roles (item finder, TMA producer, MMA issue, marks, two softmax
warpgroups, code expansion) meet on mbarriers by parity.  The model transcribes every
wait, arrival, load, MMA and commit with the kernel's phase formulas and runs
the roles under random interleavings: copies land in any order, the tensor
pipe runs in issue order.  Items have one or two sub-tiles and any number of
key tiles, none included.  Every run must end, and every access must find the
tile it expects: ring slots, Q, the marks, S, P (which overwrites S) and O.
"""
import random

import pytest

from tests.test_attn_protocol import Bar

META, WORKS = 4, 4


class Sim:
    wrong = None

    def __init__(self, items, kv8, seed, slow=None):
        self.slow = slow  # a role that seldom runs: phases that pass it by unseen show
        self.items, self.kv8, self.rnd = items, kv8, random.Random(seed)  # items: (sub-tiles, key tiles)
        self.NS = 4 if kv8 else 5
        B = {}
        for s in range(self.NS):
            B[f"raw{s}"], B[f"full{s}"], B[f"empty{s}"] = Bar(1), Bar(1), Bar(1)
        for m in range(META):
            B[f"marked{m}"] = Bar(1)
            B[f"unmarked{m}"] = Bar(1)
        for u in range(2):
            for n in ("q_raw", "q_full", "q_empty", "s", "p0", "p1", "o_full"):
                B[f"{n}{u}"] = Bar(1)
        self.b = B
        for k in range(WORKS):
            B[f"work_full{k}"], B[f"work_empty{k}"] = Bar(1), Bar(6 if kv8 else 5)
        self.works = [None] * WORKS
        self.slot = [None] * self.NS     # what a ring slot holds: (kind, item, tile, state)
        self.users = [0] * self.NS       # MMAs issued that will read it
        self.q = [None, None]
        self.qusers = [0, 0]
        self.marks = [None] * META
        self.qpow = [[None, None], [None, None]]
        self.S, self.O = [None, None], [None, None]  # S: ("S", i, j) or ("P", i, j); O: (i, tiles summed)
        self.tma, self.pipe = [], []

    def wait(self, name, n):
        while not self.b[name].done(n & 1):
            yield

    def finder(self):
        for k, item in enumerate(list(enumerate(self.items)) + [None]):
            if k >= WORKS and self.wrong != "works":
                yield from self.wait(f"work_empty{k % WORKS}", k // WORKS - 1)
            self.works[k % WORKS] = (k, item)
            self.b[f"work_full{k % WORKS}"].arrive()
            yield

    def take(self, k, keep=False):
        """The k-th item (None at the end); its place is freed at once unless kept."""
        yield from self.wait(f"work_full{k % WORKS}", k // WORKS)
        n, item = self.works[k % WORKS]
        assert n == k, "item overwritten"
        if item is not None and not keep:
            self.b[f"work_empty{k % WORKS}"].arrive()
        return item

    def producer(self):
        n, qn, work_n = 0, [0, 0], 0
        while True:
            item = yield from self.take(work_n)
            work_n += 1
            if item is None:
                return
            i, (nsub, nt) = item
            if nt == 0:
                continue
            for u in range(nsub):
                if qn[u] > 0:
                    yield from self.wait(f"q_empty{u}", qn[u] - 1)
                assert self.qusers[u] == 0
                bar = f"q_raw{u}" if self.kv8 else f"q_full{u}"
                self.b[bar].arrive(1)
                self.tma.append(("q", u, i, bar))
                qn[u] += 1
            for j in range(nt):
                for kind in "KV":
                    s = n % self.NS
                    if n >= self.NS:
                        yield from self.wait(f"empty{s}", n // self.NS - 1)
                    assert self.users[s] == 0, "slot overwritten before it was read"
                    self.slot[s] = None
                    self.b[f"raw{s}"].arrive(1)
                    self.tma.append(("slot", s, (kind, i, j), f"raw{s}"))
                    n += 1
                    yield

    def qk(self, u, n, i, j):
        s = n % self.NS
        assert self.slot[s] == ("K", i, j, "ready"), (self.slot[s], i, j)
        assert self.q[u] == i
        self.users[s] += 1
        self.qusers[u] += 1
        self.pipe.append(("qk", u, s, i, j))
        self.pipe.append(("commit", f"s{u}"))

    def mma(self):
        n, items, pn, work_n, tiles = 0, [0, 0], [0, 0], 0, 0
        while True:
            item = yield from self.take(work_n)
            work_n += 1
            if item is None:
                return
            i, (nsub, nt) = item
            if nt == 0:
                continue
            yield from self.wait(f"full{n % self.NS}", n // self.NS)
            for u in range(nsub):
                yield from self.wait(f"q_full{u}", items[u])
                self.qk(u, n, i, 0)
                if nt == 1:
                    self.pipe.append(("commit", f"q_empty{u}"))
                yield
            self.pipe.append(("commit", f"empty{n % self.NS}"))
            n += 1
            for j in range(nt):
                sv, sk, more = n, n + 1, j + 1 < nt
                yield from self.wait(f"full{sv % self.NS}", sv // self.NS)
                for u in range(nsub):
                    s = sv % self.NS
                    for half in range(2):
                        if not (self.wrong == "p" and half):
                            yield from self.wait(f"p{half}{u}", pn[u])
                        assert self.slot[s] == ("V", i, j, "ready")
                        self.users[s] += 1
                        self.pipe.append(("pv", u, s, i, j, half))
                        yield
                    pn[u] += 1
                    if u == nsub - 1:
                        self.pipe.append(("commit", f"empty{s}"))
                        if self.kv8:
                            self.pipe.append(("commit", f"unmarked{tiles % META}"))
                    if not more:
                        self.pipe.append(("commit", f"o_full{u}"))
                    yield
                    if more:
                        if u == 0:
                            yield from self.wait(f"full{sk % self.NS}", sk // self.NS)
                        self.qk(u, sk, i, j + 1)
                        if j + 2 == nt:
                            self.pipe.append(("commit", f"q_empty{u}"))
                        if u == nsub - 1:
                            self.pipe.append(("commit", f"empty{sk % self.NS}"))
                        yield
                n += 2 if more else 1
                tiles += 1
            for u in range(nsub):
                items[u] += 1

    def ready(self, s, what):
        assert self.slot[s] == what + ("raw",)
        self.slot[s] = what + ("ready",)
        self.b[f"full{s}"].arrive()

    def mark(self):
        n = tiles = work_n = 0
        while True:
            item = yield from self.take(work_n)
            work_n += 1
            if item is None:
                return
            i, (nsub, nt) = item
            for j in range(nt):
                s = n % self.NS
                if not self.kv8:
                    yield from self.wait(f"raw{s}", n // self.NS)
                elif self.wrong == "stale":  # the K before, whose barrier may be a phase further
                    if tiles > 0:
                        yield from self.wait(f"raw{(n - 2) % self.NS}", (n - 2) // self.NS)
                elif tiles >= META:
                    yield from self.wait(f"unmarked{tiles % META}", tiles // META - 1)
                self.marks[tiles % (1 if self.wrong == "meta" else META - (self.wrong == "ahead"))] = (i, j)
                if self.kv8:
                    self.b[f"marked{tiles % META}"].arrive()
                    n += 2
                else:
                    self.ready(s, ("K", i, j))
                    s = (n + 1) % self.NS
                    yield from self.wait(f"raw{s}", (n + 1) // self.NS)
                    self.ready(s, ("V", i, j))
                    n += 2
                yield
                tiles += 1

    def expand(self):
        n, tiles, qn, work_n = 0, 0, [0, 0], 0
        while True:
            item = yield from self.take(work_n)
            work_n += 1
            if item is None:
                return
            i, (nsub, nt) = item
            if nt == 0:
                continue
            for u in range(nsub):
                yield from self.wait(f"q_raw{u}", qn[u])
                assert self.q[u] == i
                self.qpow[u][qn[u] % (1 if self.wrong == "qpow" else 2)] = i
                qn[u] += 1
                self.b[f"q_full{u}"].arrive()
                yield
            for j in range(nt):
                m = tiles % META
                yield from self.wait(f"marked{m}", tiles // META)
                for kind in "KV":
                    s = n % self.NS
                    yield from self.wait(f"raw{s}", n // self.NS)
                    yield
                    assert self.marks[m] == (i, j), "scales overwritten"
                    self.ready(s, (kind, i, j))
                    n += 1
                    yield
                tiles += 1

    def softmax(self, u):
        sn = items = tiles = work_n = 0
        while True:
            item = yield from self.take(work_n, keep=True)
            if item is None:
                return
            i, (nsub, nt) = item
            if u >= nsub:
                tiles += nt
                self.b[f"work_empty{work_n % WORKS}"].arrive()
                work_n += 1
                continue
            for j in range(nt):
                yield from self.wait(f"s{u}", sn)
                assert self.S[u] == ("S", i, j), (self.S[u], i, j)
                for _ in range(3):  # the marks are read until P is complete
                    assert self.marks[tiles % (1 if self.wrong == "meta" else META - (self.wrong == "ahead"))] == (i, j), "marks overwritten"
                    yield
                if self.kv8 and j == 0:
                    assert self.qpow[u][items % (1 if self.wrong == "qpow" else 2)] == i
                if j > 0:
                    assert self.O[u] == (i, j), "O rescaled while a PV is pending"
                for half in range(2):
                    yield
                    assert self.S[u] == (("P0", i, j) if half else ("S", i, j)) or half and self.S[u] == ("P0 read", i, j)
                    self.S[u] = (f"P{half}" + (" after" if self.S[u][0] == "P0 read" else ""), i, j)
                    self.b[f"p{half}{u}"].arrive()
                sn, tiles = sn + 1, tiles + 1
                yield
            if nt:
                yield from self.wait(f"o_full{u}", items)
                items += 1
                for _ in range(2):
                    assert self.O[u] == (i, nt), (self.O[u], i, nt)
                    yield
            assert self.works[work_n % WORKS][0] == work_n, "item overwritten while in use"
            self.b[f"work_empty{work_n % WORKS}"].arrive()
            work_n += 1

    def step_tma(self):
        kind, at, what, bar = self.tma.pop(self.rnd.randrange(len(self.tma)))
        if kind == "q":
            self.q[at] = what
        else:
            self.slot[at] = what + ("raw",)
        self.b[bar].complete_tx(1)

    def step_pipe(self):
        op = self.pipe.pop(0)
        if op[0] == "commit":
            self.b[op[1]].arrive()
            return
        u, s, i, j = op[1:5]
        self.users[s] -= 1
        if op[0] == "qk":
            assert self.S[u] is None or self.S[u][0] == "done", ("S overwritten", self.S[u])
            self.S[u] = ("S", i, j)
            self.qusers[u] -= 1
        else:
            half = op[5]
            assert self.S[u][1:] == (i, j) and self.S[u][0] in (("P1", "P1 after") if half else ("P0", "P1")), self.S[u]
            if half:
                assert self.O[u] == (i, j, "half")
                self.S[u], self.O[u] = ("done", i, j), (i, j + 1)
            else:
                if j > 0:
                    assert self.O[u] == (i, j)
                self.O[u] = (i, j, "half")
                if self.S[u][0] == "P0":
                    self.S[u] = ("P0 read", i, j)

    def run(self):
        roles = [self.finder(), self.producer(), self.mma(), self.mark(), self.softmax(0), self.softmax(1)]
        if self.kv8:
            roles.append(self.expand())
        idle, slow = 0, roles[self.slow % len(roles)] if self.slow is not None else None
        while roles or self.pipe or self.tma:
            k = self.rnd.randrange(len(roles) + 2)
            if self.slow is not None and k < len(roles) and roles[k] is slow and self.rnd.random() < 0.98:
                continue  # the others run far ahead of it
            before = (len(self.tma), len(self.pipe), len(roles), tuple(b.phase * 1000 + b.pend for b in self.b.values()))
            if k < len(roles):
                try:
                    next(roles[k])
                except StopIteration:
                    roles.pop(k)
            elif k == len(roles) and self.tma:
                self.step_tma()
            elif k == len(roles) + 1 and self.pipe:
                self.step_pipe()
            after = (len(self.tma), len(self.pipe), len(roles), tuple(b.phase * 1000 + b.pend for b in self.b.values()))
            idle = idle + 1 if before == after else 0
            assert idle < (5000 if slow is None else 60000), "deadlock"


def random_items(rnd):
    return [(rnd.choice([1, 2, 2]), rnd.choice([0, 1, 1, 2, 3, 5])) for _ in range(rnd.randrange(1, 12))]


@pytest.mark.parametrize("kv8", [False, True])
def test_protocol(kv8):
    for seed in range(150):
        Sim(random_items(random.Random(seed)), kv8, seed).run()


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("slow", range(7))
def test_protocol_with_a_slow_role(kv8, slow):
    for seed in range(20):
        Sim(random_items(random.Random(seed)), kv8, seed, slow).run()


def test_a_phase_that_passes_unseen_is_caught():
    class Bad(Sim):
        wrong = "stale"

    with pytest.raises(AssertionError, match="deadlock"):
        for seed in range(40):
            Bad(random_items(random.Random(seed)), True, seed, 3).run()


@pytest.mark.parametrize("wrong", ["p", "meta", "ahead", "qpow", "works"])
def test_protocol_errors_are_caught(wrong):
    class Bad(Sim):
        pass

    Bad.wrong = wrong
    with pytest.raises(AssertionError):
        for seed in range(200):
            Bad([(2, 4), (2, 1), (1, 1), (2, 1), (2, 3), (2, 2), (1, 1)], wrong in ("qpow", "ahead"), seed).run()
