"""CPU: the barrier protocol of the chunk attention kernel, as a model of its roles run in random
orders.  An mbarrier wait names a phase by its parity alone, so a wait for phase n passes by mistake
once phase n + 1 has ended unseen; the model checks at every poll that parity and phase agree, that
no ring slot is overwritten before it is read, that a part's Q is not replaced under the MMAs that
read it, that the places of the row factors last as long as they are read, and that every run ends."""
import os
import random
import re

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "glm53_flash_dual_dgx_spark_b200", "csrc", "mla_prefill.cu")).read()


def constant(name):
    return int(re.search(rf"constexpr int {name} = (\d+);", SOURCE).group(1))


SLOTS, V_STAGES = constant("kStages"), constant("kVStages")
PLACES = int(re.search(r"64 \* \(parts & (\d)\)", SOURCE).group(1)) + 1


class Barrier:
    def __init__(self):
        self.done = 0

    def arrive(self):
        self.done += 1

    def passed(self, phase):
        by_parity = (self.done & 1) != (phase & 1)
        assert by_parity == (self.done > phase), (self.done, phase)
        return by_parity


def simulate(parts, k_stages, places, seed):
    rnd = random.Random(seed)
    empty, full, land = ([Barrier() for _ in range(SLOTS)] for _ in range(3))
    s_full, s_free = [Barrier(), Barrier()], [Barrier(), Barrier()]
    p_full, pv_done, q_full, q_free, q_land, o_free = (Barrier() for _ in range(6))
    ring, q_in, factor, flying = [None] * SLOTS, [0], [None] * places, []
    factor[0] = 0

    def stages(n):
        return n * (k_stages + V_STAGES)

    def mma():
        u = tile = 0

        def stage():
            nonlocal u
            while not full[u % SLOTS].passed(u // SLOTS):
                yield
            assert ring[u % SLOTS] == u
            full[(u + 1) % SLOTS].passed((u + 1) // SLOTS)      # the look at the next stage's barrier
            yield
            assert ring[u % SLOTS] == u
            empty[u % SLOTS].arrive()
            u += 1

        for j, n in enumerate(parts):
            while j > 0 and not q_full.passed(j - 1):
                yield
            for i in range(n + 1):
                if i < n:
                    while tile >= 2 and not s_free[tile & 1].passed((tile >> 1) - 1):
                        yield
                    for _ in range(k_stages):
                        assert q_in[0] == j
                        yield from stage()
                    s_full[tile & 1].arrive()
                    if i == n - 1:
                        q_free.arrive()
                if i > 0:
                    while not p_full.passed(tile - 1):
                        yield
                    while i == 1 and j > 0 and not o_free.passed(j - 1):
                        yield
                    for _ in range(V_STAGES):
                        yield from stage()
                    pv_done.arrive()
                tile += 1
            tile -= 1

    def softmax():
        tile = 0
        for j, n in enumerate(parts):
            for i in range(n):
                while not s_full[tile & 1].passed(tile >> 1):
                    yield
                if i == 0:
                    assert factor[j % places] == j
                s_free[tile & 1].arrive()
                yield
                while i > 0 and not pv_done.passed(tile - 1):
                    yield
                p_full.arrive()
                tile += 1
                yield
            while not pv_done.passed(tile - 1):
                yield
            o_free.arrive()
            yield

    def queries():
        for j in range(1, len(parts)):
            factor[j % places] = j
            yield
            while not q_free.passed(j - 1):
                yield
            q_in[0] = j
            q_land.arrive()
            while not q_land.passed(j - 1):
                yield
            q_full.arrive()
            yield

    def copy(mine):
        for u in range(sum(stages(n) for n in parts)):
            if u & 1 == mine:
                while u >= SLOTS and not empty[u % SLOTS].passed(u // SLOTS - 1):
                    yield
                ring[u % SLOTS] = u
                flying.append(u)
                yield

    def landing():
        while True:
            if flying:
                land[flying.pop(rnd.randrange(len(flying))) % SLOTS].arrive()
            elif len(live) == 1:
                return
            yield

    def relay():
        for u in range(sum(stages(n) for n in parts)):
            while not land[u % SLOTS].passed(u // SLOTS):
                yield
            full[u % SLOTS].arrive()
            yield

    roles = [mma(), softmax(), queries(), copy(0), copy(1), relay(), landing()]
    live = set(range(len(roles)))
    speed = [rnd.choice([1, 1, 5, 40]) for _ in roles]
    idle = 0
    while live:
        order = sorted(live)
        k = rnd.choices(order, [speed[i] for i in order])[0]
        try:
            next(roles[k])
        except StopIteration:
            live.discard(k)
            idle = 0
        idle += 1
        assert idle < 300000, "no progress"


def random_parts(seed):
    r = random.Random(seed)
    return [r.choice([1, 1, 2, 4]) for _ in range(r.randint(1, 8))]


@pytest.mark.parametrize("k_stages", [8, 9])
def test_every_wait_is_for_its_phase(k_stages):
    for seed in range(60):
        simulate(random_parts(seed), k_stages, PLACES, seed)


def test_fewer_places_for_the_factors_would_not_do():
    with pytest.raises(AssertionError):
        for seed in range(400):
            simulate([1] * 8, 8, PLACES // 2, seed)
