"""GPU: giving pages back where positions are near the largest of an int (a page of one token has as many
pages as tokens)."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_extend_pages_gpu import Model, ints, same

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("page", [1, 2, 16])
@pytest.mark.parametrize("sinks", [MOST - 300, MOST - 255, MOST - 1, MOST, 2 ** 40])
def test_sinks_past_every_sequence(page, sinks):
    """Every token is one of the first: nothing is behind the window, and what lies past the end goes."""
    m = Model(4, 400, page, 900, seed=page)
    for s, n in enumerate([0, 1, 300 * page + 1, 390 * page]):
        m.fill(s, n)
    m.seq[3] = 370 * page
    dev = m.cuda()
    m.trim([0, 1, 2, 3], 5, sinks)
    rt.trim_pages(dev[0], dev[1], ints([0, 1, 2, 3]), dev[2], page, window=5, sinks=sinks)
    assert rt.device_errors() == m.error == 0
    assert not bool((dev[0] == _lib.PAGE_TRIMMED).any()) and int((dev[0][3] >= 0).sum()) == 370
    same(m, dev)


@pytest.mark.parametrize("length", [MOST - 255, MOST])
def test_a_length_that_no_table_holds(length):
    """Behind the window is then the whole table."""
    m = Model(2, 300, 1, 700, seed=2)
    for s in range(2):
        m.fill(s, 300)
    m.seq[1] = length
    dev = m.cuda()
    for window, sinks in ((0, 0), (7, 290)):
        m.trim([1, 0], window, sinks)
        rt.trim_pages(dev[0], dev[1], ints([1, 0]), dev[2], 1, window=window, sinks=sinks)
        assert rt.device_errors() == m.error == 0
        same(m, dev)
    assert bool((dev[0][1, 290:] == _lib.PAGE_TRIMMED).all()) and torch.equal(dev[0][1, :290], m.tables[1, :290].cuda())
