"""CPU: the form of the chunk attention kernel whose Q warps copy Q straight into its operand and tell the
MMA warp of the next part (queries of several units in a window), as the model of test_prefill_operands
with those two roles, and the MMA warp's wait for the output of the part before, as mla_prefill.cu has
them there: a change of a wait, an arrival or a role has to be made here too.

The number of the next part's tiles goes through two words, written before the arrival that says its Q is
there; 0 after the last part, once its last QK is done."""
import pytest

from test_prefill_operands import CTAS, K_STAGES, Q_AGENTS, SLOTS, V_STAGES, Broken, Model, need, random_parts


class Direct(Model):
    def __init__(self, parts, seed, without=()):
        super().__init__(parts, seed, without)
        self.told = [None, None]
        self.copied = [0, 0]
        self.scratch = None

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

        j, n = 0, self.parts[0]
        while n > 0:
            for i in range(n + 1):
                if i == 1 and j > 0:
                    yield from self.wait("O_FREE", self.o_free, j - 1)
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
                    for k in range(V_STAGES):
                        yield from stage("pv", j, tile - 1, i == 1 and k == 0)

                    def summed(j=j, i=i):
                        for c in CTAS:
                            self.o[c] = (j, i)
                            self.pv_done[c].arrive()
                    self.pipe.append(("commit", summed))
                tile += 1
            tile -= 1
            j += 1
            yield from self.wait("Q_FULL", self.q_full, j - 1)
            n = self.told[j & 1]
            need(n == (self.parts[j] if j < len(self.parts) else 0), "told", j, n)
            yield
        need(j == len(self.parts), "parts", j)
        self.posted, self.live_mma = True, False

    def queries(self, c, agent):
        for j in range(1, len(self.parts)):
            yield from self.wait("Q_FREE", self.q_free[c], j - 1)
            self.q[c] = None                                 # (the agents' rows land one by one)
            yield
            self.copied[c] += 1
            while self.copied[c] < len(Q_AGENTS) * j:        # the agents' own barrier
                yield
            self.q[c] = j
            if agent == 0:
                if c == 0:
                    self.told[j & 1] = self.parts[j]
                    yield
                self.q_full.arrive()
            yield
        yield from self.wait("Q_FREE at the end", self.q_free[c], len(self.parts) - 1)
        if agent == 0:
            if c == 0:
                self.told[len(self.parts) & 1] = 0
                yield
            self.q_full.arrive()


def test_no_operand_is_touched_too_early():
    for seed in range(20):
        Direct(random_parts(seed), seed).run()
    Direct([1], 0).run()


@pytest.mark.parametrize("name", ["FULL", "EMPTY", "LAND", "S_FULL", "P_FULL", "Q_FULL", "Q_FREE", "Q_FREE at the end", "PV_DONE before P",
                                  "PV_DONE before the output"])
def test_without_one_wait_some_order_breaks_a_rule(name):
    with pytest.raises((Broken, TypeError)):
        for seed in range(200):
            Direct(random_parts(seed), seed, (name,)).run()
