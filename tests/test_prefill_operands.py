"""CPU: who may touch which operand of the chunk attention kernel, and when, as a model of its roles run
in random orders.  The model is written by hand after mla_prefill.cu: a change of a wait, an arrival or
a role there has to be made here too.

Two CTAs; the tensor pipe takes MMAs in the order of their issue and runs each for a while.  At the
start and at the end of each it must find the Q of its part, the stage of its number, P of its tile,
and S and O that nobody else reads or writes; a commit arrives when all MMAs before it are done.  The
scratch of a part's Q must be whole and unchanged while it is copied.  Each wait that the others do not
imply is left out in turn, and some order then breaks a rule."""
import os
import random
import re

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "glm53_flash_dual_dgx_spark_b200", "csrc", "mla_prefill.cu")).read()


def constant(name):
    return int(re.search(rf"constexpr int {name} = (\d+);", SOURCE).group(1))


SLOTS, V_STAGES, K_STAGES = constant("kStages"), constant("kVStages"), 8
PER_TILE = K_STAGES + V_STAGES
CTAS, Q_AGENTS = (0, 1), (0, 1)      # (agent 0 of a CTA's Q warps issues the copy)


class Broken(AssertionError):
    pass


def need(ok, *what):
    if not ok:
        raise Broken(*what)


class Barrier:
    def __init__(self, arrivals=1):
        self.arrivals, self.count, self.done = arrivals, 0, 0

    def arrive(self):
        self.count += 1
        if self.count == self.arrivals:
            self.count, self.done = 0, self.done + 1

    def passed(self, phase):
        by_parity = (self.done & 1) != (phase & 1)
        need(by_parity == (self.done > phase), "parity", self.done, phase)
        return by_parity


class Model:
    def __init__(self, parts, seed, without=()):
        self.parts, self.rnd, self.without = parts, random.Random(seed), without
        two = lambda n=1: [[Barrier(n) for _ in range(SLOTS)] for _ in CTAS]  # noqa: E731
        self.full = [Barrier(2) for _ in range(SLOTS)]
        self.empty, self.land = two(), two()
        self.s_full = [[Barrier(), Barrier()] for _ in CTAS]
        self.s_free = [Barrier(2), Barrier(2)]
        self.p_full, self.q_full, self.o_free = Barrier(2), Barrier(2), Barrier(2)
        self.pv_done, self.q_free, self.q_land = ([Barrier() for _ in CTAS] for _ in range(3))
        self.ring = [[None] * SLOTS for _ in CTAS]
        self.q, self.p, self.scratch = [0, 0], [None, None], [[None, None], [None, None]]
        self.s, self.s_read = [[None, None], [None, None]], [[True, True], [True, True]]
        self.o, self.o_busy = [None, None], [False, False]      # (part, tiles summed); softmax at work on it
        self.pipe, self.flying = [], []
        self.written, self.posted = [0, 0], False

    def wait(self, name, barrier, phase):
        while name not in self.without and not barrier.passed(phase):
            yield

    # -------------------------------------------------------------- tensor pipe
    def operands(self, op):
        kind, j, tile, stage, first = op
        for c in CTAS:
            need(self.ring[c][stage % SLOTS] == stage, "stage", op)
            if kind == "qk":
                need(self.q[c] == j, "Q", op)
            else:
                need(self.p[c] == tile, "P", op, self.p)
                need(not self.o_busy[c], "O", op)

    def tensor(self):
        while True:
            if not self.pipe:
                if self.posted and not self.live_mma:
                    return
                yield
                continue
            op = self.pipe[0]
            if op[0] == "commit":
                op[1]()
            else:
                kind, j, tile, stage, first = op
                if kind == "qk" and first:
                    for c in CTAS:
                        need(self.s_read[c][tile & 1], "S", op)
                        self.s[c][tile & 1], self.s_read[c][tile & 1] = None, False
                if kind == "pv" and first:
                    for c in CTAS:
                        need(self.o[c] is None or self.o[c][0] == j, "O of the last part", op)
                self.operands(op)
                for _ in range(self.rnd.randint(1, 3)):
                    yield
                self.operands(op)
            self.pipe.pop(0)
            yield

    def mma(self):
        u = tile = 0
        self.live_mma = True

        def both(barriers):
            return lambda: [b.arrive() for b in barriers]

        def stage(kind, j, t, first):
            nonlocal u
            yield from self.wait("FULL", self.full[u % SLOTS], u // SLOTS)
            self.pipe.append((kind, j, t, u, first))
            self.pipe.append(("commit", both([self.empty[c][u % SLOTS] for c in CTAS])))
            u += 1
            yield

        for j, n in enumerate(self.parts):
            if j > 0:
                yield from self.wait("Q_FULL", self.q_full, j - 1)
            for i in range(n + 1):
                if i < n:
                    if tile >= 2:
                        yield from self.wait("S_FREE", self.s_free[tile & 1], (tile >> 1) - 1)
                    for k in range(K_STAGES):
                        yield from stage("qk", j, tile, k == 0)

                    def scored(t=tile):
                        for c in CTAS:
                            self.s[c][t & 1] = t
                            self.s_full[c][t & 1].arrive()
                    self.pipe.append(("commit", scored))
                    if i == n - 1:
                        self.pipe.append(("commit", both(self.q_free)))
                if i > 0:
                    yield from self.wait("P_FULL", self.p_full, tile - 1)
                    if i == 1 and j > 0:
                        yield from self.wait("O_FREE", self.o_free, j - 1)
                    for k in range(V_STAGES):
                        yield from stage("pv", j, tile - 1, i == 1 and k == 0)

                    def summed(j=j, i=i):
                        for c in CTAS:
                            self.o[c] = (j, i)
                            self.pv_done[c].arrive()
                    self.pipe.append(("commit", summed))
                tile += 1
            tile -= 1
        self.posted, self.live_mma = True, False

    # -------------------------------------------------------------- softmax and epilogue
    def softmax(self, c):
        tile = 0
        for j, n in enumerate(self.parts):
            for i in range(n):
                yield from self.wait("S_FULL", self.s_full[c][tile & 1], tile >> 1)
                for _ in range(2):
                    need(self.s[c][tile & 1] == tile, "S read", j, i)
                    yield
                self.s_read[c][tile & 1] = True
                self.s_free[tile & 1].arrive()
                yield
                if i > 0:
                    yield from self.wait("PV_DONE before P", self.pv_done[c], tile - 1)
                    self.o_busy[c] = True                  # O scaled to a new maximum
                    need(self.o[c] == (j, i), "O scaled", j, i, self.o)
                    yield
                    self.o_busy[c] = False
                self.p[c] = None
                yield
                self.p[c] = tile
                self.p_full.arrive()
                tile += 1
                yield
            yield from self.wait("PV_DONE before the output", self.pv_done[c], tile - 1)
            self.o_busy[c] = True
            for _ in range(3):
                need(self.o[c] == (j, n), "O stored", j, self.o)
                yield
            self.o_busy[c], self.o[c] = False, None
            self.o_free.arrive()
            yield

    # -------------------------------------------------------------- Q of the next parts
    def queries(self, c, agent):
        for j in range(1, len(self.parts)):
            need(("q", c) not in [f[:2] for f in self.flying], "scratch under its copy", j)
            self.scratch[c][agent] = None
            yield
            self.scratch[c][agent] = j
            self.written[c] += 1
            while self.written[c] < len(Q_AGENTS) * j:      # the agents' own barrier
                yield
            yield from self.wait("Q_FREE", self.q_free[c], j - 1)
            if agent == 0:
                need(self.scratch[c] == [j, j], "scratch", self.scratch[c], j)
                self.flying.append(("q", c, j))
                yield
            yield from self.wait("Q_LAND", self.q_land[c], j - 1)
            if agent == 0:
                self.q_full.arrive()
            yield

    # -------------------------------------------------------------- ring
    def copy(self, c, mine):
        for u in range(sum(self.parts) * PER_TILE):
            if u & 1 != mine:
                continue
            if u >= SLOTS:
                yield from self.wait("EMPTY", self.empty[c][u % SLOTS], u // SLOTS - 1)
                yield
            self.ring[c][u % SLOTS] = None
            self.flying.append(("stage", c, u))
            if u >= SLOTS:                                 # (the first stages are copied before the roles begin)
                yield

    def landing(self):
        while self.flying or self.busy > 1:
            if self.flying:
                kind, c, x = self.flying[k := self.rnd.randrange(len(self.flying))]
                if kind == "q":
                    need(self.scratch[c] == [x, x], "scratch under its copy", x)
                    self.q[c] = x
                    self.q_land[c].arrive()
                else:
                    self.ring[c][x % SLOTS] = x
                    self.land[c][x % SLOTS].arrive()
                self.flying.pop(k)
            yield

    def relay(self, c):
        for u in range(sum(self.parts) * PER_TILE):
            yield from self.wait("LAND", self.land[c][u % SLOTS], u // SLOTS)
            self.full[u % SLOTS].arrive()
            yield

    def run(self):
        roles = [self.mma(), self.tensor(), self.landing()]
        for c in CTAS:
            roles += [self.softmax(c), self.copy(c, 0), self.copy(c, 1), self.relay(c)] + [self.queries(c, a) for a in Q_AGENTS]
        self.live_mma = True
        live = dict(enumerate(roles))
        speed = [self.rnd.choice([1, 1, 5, 40]) for _ in roles]
        steps = stalled = 0
        while live:
            self.busy = len(live)
            if steps % 500 == 0:                           # one of them falls far behind for a while
                stalled = self.rnd.randrange(len(roles))
            keys = [i for i in live if i != stalled] or list(live)
            k = self.rnd.choices(keys, [speed[i] for i in keys])[0]
            try:
                next(live[k])
            except StopIteration:
                del live[k]
                steps = 0
            steps += 1
            need(steps < 300000, "no progress")


def random_parts(seed):
    r = random.Random(seed)
    return [r.choice([1, 1, 2, 3]) for _ in range(r.randint(2, 5))]


def test_no_operand_is_touched_too_early():
    for seed in range(20):
        Model(random_parts(seed), seed).run()


@pytest.mark.parametrize("name", ["FULL", "EMPTY", "LAND", "S_FULL", "P_FULL", "Q_FULL", "Q_FREE", "Q_LAND", "PV_DONE before P",
                                  "PV_DONE before the output"])
def test_without_one_wait_some_order_breaks_a_rule(name):
    with pytest.raises(Broken):
        for seed in range(200):
            Model(random_parts(seed), seed, (name,)).run()


@pytest.mark.parametrize("name", ["S_FREE", "O_FREE"])
def test_waits_that_the_order_of_the_others_implies(name):
    """P of a tile arrives after S of the tile and O of the part before it were read, and the MMAs that
    would overwrite those are issued behind the wait for P."""
    for seed in range(8):
        Model(random_parts(seed), seed, (name,)).run()
