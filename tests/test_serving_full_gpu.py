"""GPU: the serving loop stops when its cache is full, and goes on where its last page is just enough."""
import pytest

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from glm53_flash_dual_dgx_spark_b200 import serving_step

pytestmark = pytest.mark.gpu


class Small(serving_step.Cache):
    """A cache of so many pages, whatever the loop asks for."""

    pages = 0

    def __init__(self, num_pages, *args):
        super().__init__(self.pages, *args)


# a prompt of 130 tokens (3 pages) and one of 65 (2), then four forks with a last page of their own each (9), which at
# 130 + 63 tokens need another each, as the first prompt does (14), while the second one's 128 do not; with a window of 20 no
# sequence keeps more than two pages (12)
@pytest.mark.parametrize("pages,steps,window", [(4, 3, 0), (8, 3, 0), (9, 62, 0), (9, 63, 0), (13, 63, 0), (14, 63, 0), (12, 200, 20)])
def test_a_full_cache_stops_the_loop(pages, steps, window, monkeypatch):
    monkeypatch.setattr(serving_step, "Cache", Small)
    monkeypatch.setattr(Small, "pages", pages)
    run = lambda: serving_step.run(heads=2, prompt=130, steps=steps, window=window, chunk=64)  # noqa: E731
    need = 9 if steps <= 62 else 14
    if pages >= need or window:
        got = run()
        assert got["device_errors"] == 0 and got["fork_equals_parent"] and got["compaction_keeps_outputs"]
    else:
        with pytest.raises(RuntimeError, match="full"):
            run()
        assert rt.device_errors() & _lib.DEVERR_CAPACITY
