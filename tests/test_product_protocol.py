"""The barriers of the projection's tcgen05 kernel (csrc/linear_tc.cuh) as a model on the CPU: its roles as coroutines that a random scheduler interleaves, asynchronous copies,
products and stores that end at any later time.  Every chunk must be stored once, with its own tile's finished sum and its own residual, and nothing may wait for good."""
import random

import pytest


class Bar:
    """mbarrier: a phase ends when `count` arrivals are in and no bytes are outstanding."""

    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def _check(self):
        if self.pending == 0 and self.tx == 0:
            self.pending, self.phase = self.count, self.phase ^ 1

    def arrive(self, tx=0):
        assert self.pending > 0, "an arrival too many"
        self.pending -= 1
        self.tx += tx
        self._check()

    def complete(self, n=1):
        self.tx -= n
        self._check()

    def passed(self, parity):
        return self.phase != parity


class Chunks:
    """Chunks of 64 columns of a CTA's tiles that one warpgroup owns (linear_tc.cuh: Walk, Chunks)."""

    def __init__(self, cfg, unit, wg):
        self.cfg, self.wg, self.item, self.first, self.c = cfg, wg, unit, 0, wg

    def next_tile(self):
        self.item += self.cfg["units"]
        if not self.cfg["slope"]:
            self.first = (self.first + self.cfg["chunks"]) % self.cfg["G"]
        self.c = self.wg - self.first + (self.cfg["G"] if self.wg < self.first else 0)

    def in_tile(self):      # the last column of tiles is narrower
        cfg = self.cfg
        return self.c < (cfg["last_chunks"] if self.item % cfg["tiles_n"] == cfg["tiles_n"] - 1 else cfg["chunks"])

    def find(self):
        while self.item < self.cfg["items"]:
            if self.in_tile():
                return True
            self.next_tile()
        return False

    def take(self):
        self.c += self.cfg["G"]


class Model:
    def __init__(self, cfg, rng):
        self.cfg, self.rng = cfg, rng
        self.ranks = 2 if cfg["pair"] else 1
        self.stored, self.actors = {}, []
        for unit in range(cfg["units"]):
            self.add_unit(unit)

    def add_unit(self, unit):
        cfg, R = self.cfg, self.ranks
        S, G = cfg["stages"], cfg["G"]
        u = dict(full=[Bar(1) for _ in range(S)], free=[Bar(G * R) for _ in range(2)], queue=[], acc=[None, None], reads=[0, 0],
                 cta=[dict(empty=[Bar(1) for _ in range(S)], ready=[Bar(1) for _ in range(2)], ring=[None] * S, avail=[Bar(1) for _ in range(2 * G)],
                           done=[Bar(1) for _ in range(2 * G)], buf=[None] * (2 * G)) for _ in range(R)])
        self.actors += [self.issuer(u, unit), self.tensor(u)]
        for r in range(R):
            self.actors.append(self.producer(u, unit, r))
            for g in range(G):
                self.actors += [self.mover(u, unit, r, g), self.epilogue(u, unit, r, g)]

    def later(self, act):      # an asynchronous operation that ends at some time
        def run():
            for _ in range(self.rng.randrange(6)):
                yield None
            act()
        self.actors.append(run())

    # ---------------------------------------------------------------- roles
    def producer(self, u, unit, r):
        cfg, cta, st, ph = self.cfg, u["cta"][r], 0, 1
        for item in range(unit, cfg["items"], cfg["units"]):
            for kb in range(cfg["steps"]):
                yield lambda: cta["empty"][st].passed(ph)
                if r == 0:
                    u["full"][st].arrive(tx=self.ranks)

                def land(st=st, what=(item, kb)):
                    cta["ring"][st] = what
                    u["full"][st].complete()
                self.later(land)
                st += 1
                if st == cfg["stages"]:
                    st, ph = 0, ph ^ 1
                yield None

    def issuer(self, u, unit):
        cfg, st, ph, acc, acc_ph = self.cfg, 0, 0, 0, 1
        for item in range(unit, cfg["items"], cfg["units"]):
            yield lambda: u["free"][acc].passed(acc_ph)
            for kb in range(cfg["steps"]):
                yield lambda: u["full"][st].passed(ph)
                u["queue"].append(("product", acc, st, item, kb))
                u["queue"].append(("empty", st))
                st += 1
                if st == cfg["stages"]:
                    st, ph = 0, ph ^ 1
                yield None
            u["queue"].append(("ready", acc))
            acc ^= 1
            if acc == 0:
                acc_ph ^= 1
        u["queue"].append(("end",))

    def tensor(self, u):
        """Products and commits, in order, at any time after they were issued."""
        while True:
            yield lambda: bool(u["queue"])
            op = u["queue"].pop(0)
            if op[0] == "end":
                return
            if op[0] == "product":
                _, acc, st, item, kb = op
                assert all(cta["ring"][st] == (item, kb) for cta in u["cta"]), "operands of another step"
                assert kb == 0 or u["acc"][acc] == (item, kb), "sum of another tile"
                u["acc"][acc] = (item, kb + 1)
            else:
                for cta in u["cta"]:
                    (cta["empty"][op[1]] if op[0] == "empty" else cta["ready"][op[1]]).arrive()
            yield None

    def mover(self, u, unit, r, g):
        cfg, cta = self.cfg, u["cta"][r]
        head, tail = Chunks(cfg, unit, g), Chunks(cfg, unit, g)

        def prepare(b):
            i, what = 2 * g + b, ("residual", head.item, head.c, r)
            if cfg["reads"]:
                cta["avail"][i].arrive(tx=1)

                def land():
                    cta["buf"][i] = what
                    cta["avail"][i].complete()
                self.later(land)
            else:
                cta["avail"][i].arrive()
            head.take()

        for b in range(2):
            if head.find():
                prepare(b)
        ph = b = 0
        while tail.find():
            i = 2 * g + b
            yield lambda: cta["done"][i].passed(ph)
            what = cta["buf"][i]
            assert what == ("result", tail.item, tail.c, r), (what, tail.item, tail.c)
            for _ in range(self.rng.randrange(4)):      # the store reads the buffer
                yield None
            assert cta["buf"][i] == what, "written while it is stored"
            self.stored[what] = self.stored.get(what, 0) + 1
            if head.find():
                prepare(b)
            ph ^= b
            b ^= 1
            tail.take()
            yield None

    def epilogue(self, u, unit, r, g):
        cfg, cta, own = self.cfg, u["cta"][r], Chunks(self.cfg, unit, g)
        acc = ph = seq = 0
        while own.item < cfg["items"]:
            yield lambda: cta["ready"][acc].passed(ph)
            while own.in_tile():
                i = 2 * g + (seq & 1)
                yield lambda: cta["avail"][i].passed(seq >> 1 & 1)
                assert not cfg["reads"] or cta["buf"][i] == ("residual", own.item, own.c, r), "residual of another chunk"
                assert u["acc"][acc] == (own.item, cfg["steps"]), "an unfinished sum, or another tile's"
                yield None
                assert u["acc"][acc] == (own.item, cfg["steps"]), "overwritten while it is read"
                cta["buf"][i] = ("result", own.item, own.c, r)
                cta["done"][i].arrive()
                seq += 1
                own.take()
                yield None
            u["free"][acc].arrive()
            acc ^= 1
            if acc == 0:
                ph ^= 1
            own.next_tile()

    def run(self):
        waiting = [(a, None) for a in self.actors]
        self.actors = []
        while waiting:
            ready = [k for k, (_, cond) in enumerate(waiting) if cond is None or cond()]
            assert ready, "everything waits"
            k = self.rng.choice(ready)
            actor, _ = waiting[k]
            try:
                waiting[k] = (actor, next(actor))
            except StopIteration:
                waiting.pop(k)
            waiting += [(a, None) for a in self.actors]
            self.actors = []


def expected(cfg):
    ranks = 2 if cfg["pair"] else 1
    out = {}
    for item in range(cfg["items"]):
        last = item % cfg["tiles_n"] == cfg["tiles_n"] - 1
        for c in range(cfg["last_chunks"] if last else cfg["chunks"]):
            for r in range(ranks):
                out[("result", item, c, r)] = 1
    return out


# tiles of 64, 128, 192 and 256 columns; rings and warpgroups as they are built and smaller; fewer tiles than CTAs, one step of k
@pytest.mark.parametrize("chunks,G,stages,steps", [(1, 2, 8, 1), (2, 2, 4, 3), (3, 3, 4, 6), (3, 2, 5, 5), (4, 3, 3, 2), (4, 2, 2, 7), (2, 3, 1, 3)])
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("reads", [False, True])
def test_every_chunk_is_stored_once_and_nothing_waits_for_good(chunks, G, stages, steps, pair, reads):
    for seed in range(4):
        rng = random.Random(1000 * seed + chunks + 10 * G)
        tiles_n = rng.choice([1, 2, 3])
        cfg = dict(chunks=chunks, last_chunks=rng.randint(1, chunks), tiles_n=tiles_n, items=tiles_n * rng.randint(1, 4), units=rng.choice([1, 2]), G=G, stages=stages,
                   steps=steps, pair=pair, reads=reads, slope=False)
        m = Model(cfg, rng)
        m.run()
        assert m.stored == expected(cfg)


@pytest.mark.parametrize("chunks", [2, 3])
@pytest.mark.parametrize("pair", [False, True])
def test_slope_gives_a_warpgroup_the_same_chunk_of_every_tile(chunks, pair):
    rng = random.Random(chunks)
    cfg = dict(chunks=chunks, last_chunks=1, tiles_n=2, items=8, units=2, G=3, stages=4, steps=3, pair=pair, reads=True, slope=True)
    m = Model(cfg, rng)
    m.run()
    assert m.stored == expected(cfg)


def test_the_model_finds_a_missing_wait(monkeypatch):
    """Waits that now and then pass too early: the model notices."""
    passed, found = Bar.passed, 0
    for seed in range(20):
        rng = random.Random(seed)
        monkeypatch.setattr(Bar, "passed", lambda self, parity: passed(self, parity) or rng.random() < 0.02)
        try:
            Model(dict(chunks=2, last_chunks=2, tiles_n=1, items=6, units=1, G=2, stages=2, steps=2, pair=False, reads=True, slope=False), rng).run()
        except AssertionError:
            found += 1
    assert found > 10
