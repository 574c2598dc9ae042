"""GPU: a NaN in a token reaches exactly the rows that see the token, wherever the work over the
context is cut among CTA pairs: alone in its tile, in a tile of nothing else, and in a tile whose other
scores are so far below the rest that its weight is zero."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_gpu import Problem

pytestmark = pytest.mark.gpu
TILE = 256
OTHERS = [([], []), ([1, 1], [700, 3000]), ([40, 1, 3], [900, 20, 4100])]


def poison(p, b, tokens):
    """A NaN scale in each of the sequence's tokens."""
    slot = p.slots(b)[torch.as_tensor(tokens)]
    p.pool.view(-1, 288)[slot.cuda(), 256 + 9] = 0x7F


def check(p, first_nan):
    """The rows of sequence 0 from new token `first_nan` on are NaN in out and lse, no others are."""
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
    want = torch.zeros(sum(p.new), dtype=torch.bool)
    want[first_nan:p.new[0]] = True
    assert torch.equal(torch.isnan(out.float()).all(-1).all(-1).cpu(), want)
    assert torch.equal(torch.isnan(lse).all(-1).cpu(), want)
    assert not torch.isnan(out[~want.cuda()].float()).any() and not torch.isnan(lse[~want.cuda()]).any()


@pytest.mark.parametrize("others", OTHERS)
@pytest.mark.parametrize("new,H", [(1, 16), (1, 64), (3, 20), (70, 5)])
def test_newest_token_alone_in_the_last_tile(new, H, others):
    p = Problem([new, *others[0]], [20 * TILE + 1, *others[1]], H, 64, True, seed=new + H)
    poison(p, 0, [20 * TILE])
    check(p, new - 1)


@pytest.mark.parametrize("others", OTHERS)
@pytest.mark.parametrize("tile", [0, 7, 18])
@pytest.mark.parametrize("new,H", [(1, 16), (6, 33)])
def test_tile_of_nothing_but_nans(new, H, tile, others):
    p = Problem([new, *others[0]], [20 * TILE - 3, *others[1]], H, 64, True, seed=tile)
    poison(p, 0, range(tile * TILE, (tile + 1) * TILE))
    check(p, 0)


@pytest.mark.parametrize("others", OTHERS)
@pytest.mark.parametrize("tile", [0, 11, 19])
def test_tile_far_below_the_others(tile, others):
    """Scores of the tile lie about 440 (log2) below the rest: its weight underflows, its NaN does not."""
    p = Problem([2, *others[0]], [20 * TILE, *others[1]], 16, 64, False, seed=3)
    d = torch.randn(512, generator=torch.Generator().manual_seed(4))
    p.q[:2] = torch.cat([d, torch.zeros(64)]).to(torch.bfloat16).cuda()
    p.scale = 0.2
    slot = p.slots(0)[tile * TILE:(tile + 1) * TILE]
    rt.write_nvfp4((-3.0 * d).expand(TILE, 512).to(torch.bfloat16).cuda(), p.pool, slot.cuda())
    poison(p, 0, [tile * TILE + 5])
    check(p, 0)


def test_queries_that_are_nan():
    """Every row with a NaN query is NaN, and no other."""
    p = Problem([3], [20 * TILE], 4, 64, True, seed=5)
    p.q[1, 2, 40], p.q[2, 0, 530] = float("nan"), float("nan")
    out, lse = p.run()
    want = torch.zeros(3, 4, dtype=torch.bool)
    want[1, 2] = want[2, 0] = True
    assert torch.equal(torch.isnan(out.float()).all(-1).cpu(), want) and torch.equal(torch.isnan(lse).cpu(), want)
    assert not torch.isnan(out[~want.cuda()].float()).any()
