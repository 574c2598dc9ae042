"""CPU: what the bulk page copy waits for before it ends after a timed-out wait, as a model of its ring.
Piece i uses stage i % STAGES; its load is issued AHEAD pieces before it is waited for.  A wait names a
phase by its parity alone: it passes once the phase has ended and the next one has not."""
import os
import re

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "glm53_flash_dual_dgx_spark_b200", "csrc", "cache_pages.cu")).read()
STAGES = int(re.search(r"constexpr int kCopyStages = (\d+)", SOURCE).group(1))
AHEAD = STAGES // 2


def ring(mine, stuck):
    """The ring when the load of piece `stuck` does not land in time: phases ended of each stage's barrier,
    and the pieces in flight."""
    ended, issued = [0] * STAGES, list(range(min(AHEAD, mine)))
    for i in range(mine):
        if i == stuck:
            break
        ended[i % STAGES] += 1
        if i + AHEAD < mine:
            issued.append(i + AHEAD)
    return ended, [i for i in issued if i >= stuck]


def by_piece(mine, stuck):
    """(stage, parity) of each wait: the pieces in flight, each in its round's phase."""
    return [(i % STAGES, (i // STAGES) & 1) for i in range(stuck, min(stuck + AHEAD, mine))]


def by_stage(mine, stuck):
    """Every stage that was ever loaded, in the stuck piece's phase."""
    return [(s, (stuck // STAGES) & 1) for s in range(min(STAGES, mine, stuck + AHEAD))]


def covered(waits, ended, flying):
    """Whether the waits end only when all pieces in flight have landed, and all of them end then."""
    waiting = {(s, p) for s, p in waits if (ended[s] & 1) == p}      # (the others pass at once)
    landed = list(ended)
    for i in flying:
        landed[i % STAGES] += 1
    return waiting == {(i % STAGES, (i // STAGES) & 1) for i in flying} and all((landed[s] & 1) != p for s, p in waits)


@pytest.mark.parametrize("mine", [1, 3, AHEAD, STAGES, STAGES + 1, 5 * STAGES + 3])
def test_the_loads_in_flight_are_awaited_and_nothing_else(mine):
    for stuck in range(mine):
        assert covered(by_piece(mine, stuck), *ring(mine, stuck)), stuck


def test_the_kernel_waits_by_piece():
    assert re.search(r"for \(int64_t i = done; i < done \+ kAhead && i < mine; \+\+i\) "
                     r"mbar_drain_wait\(smem_u32\(&bars\[i % kCopyStages\]\), \(i / kCopyStages\) & 1\);", SOURCE)
    assert re.search(r"constexpr int kAhead = kCopyStages / 2;", SOURCE)


def test_one_phase_for_all_stages_would_not_do():
    mine = 5 * STAGES
    bad = [k for k in range(mine) if not covered(by_stage(mine, k), *ring(mine, k))]
    assert len(bad) > mine // 2
